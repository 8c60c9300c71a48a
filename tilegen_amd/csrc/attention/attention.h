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

// An operand as a call describes it: `size` elements along each axis, `stride` elements apart.
struct Operand {
  const char* name;
  const void* at;
  int axes;
  int64_t size[4], stride[4];
};

inline bool same(const Operand& x, const Operand& y) {
  bool yes = x.at == y.at && x.axes == y.axes;
  for (int i = 0; yes && i < x.axes; ++i)
    yes = x.size[i] == y.size[i] && (x.size[i] <= 1 || x.stride[i] == y.stride[i]);
  return yes;
}

// Whether two operands have a byte in common: whether the distance between them is a sum of steps
// along their axes.  Steps of one length count together; from the longest on, each number of
// them is tried that the shorter ones can make up for, which is two or three where one axis lies
// inside the next, as in slices of one array.  Layouts that need many trials count as sharing.
class Sharing {
 public:
  Sharing(const Operand& x, const Operand& y, int bytes) {
    empty_ = !x.at || !y.at;
    add(x, bytes, 1);
    add(y, bytes, -1);
    step(1, -(bytes - 1), bytes - 1);
    for (int i = 1; i < n_; ++i)    // the longest first
      for (int j = i; j && steps_[j].length > steps_[j - 1].length; --j) {
        const Step other = steps_[j];
        steps_[j] = steps_[j - 1];
        steps_[j - 1] = other;
      }
    for (int i = n_; i--;) {
      least_[i] = least_[i + 1] + steps_[i].length * steps_[i].least;
      most_[i] = most_[i + 1] + steps_[i].length * steps_[i].most;
    }
    distance_ = static_cast<Wide>(reinterpret_cast<uintptr_t>(y.at)) -
                static_cast<Wide>(reinterpret_cast<uintptr_t>(x.at));
  }
  bool operator()() {
    return !empty_ && distance_ >= least_[0] && distance_ <= most_[0] && reach(0, distance_);
  }

 private:
  using Wide = __int128;
  struct Step {
    Wide length, least, most;   // how often it may be taken
  };
  void step(Wide length, Wide least, Wide most) {
    if (length == 0) return;
    if (length < 0) {
      const Wide from = -most;
      length = -length;
      most = -least;
      least = from;
    }
    for (int i = 0; i < n_; ++i)
      if (steps_[i].length == length) {
        steps_[i].least += least;
        steps_[i].most += most;
        return;
      }
    steps_[n_++] = {length, least, most};
  }
  void add(const Operand& x, int bytes, int sign) {
    for (int i = 0; i < x.axes; ++i) {
      if (x.size[i] < 1) empty_ = true;
      const Wide last = x.size[i] - 1;
      step(static_cast<Wide>(x.stride[i]) * bytes, sign < 0 ? -last : 0, sign < 0 ? 0 : last);
    }
  }
  static Wide down(Wide n, Wide d) { return n / d - (n % d < 0); }
  bool reach(int i, Wide left) {
    if (i == n_) return left == 0;
    const Step& s = steps_[i];
    Wide from = -down(most_[i + 1] - left, s.length), to = down(left - least_[i + 1], s.length);
    if (from < s.least) from = s.least;
    if (to > s.most) to = s.most;
    for (Wide n = from; n <= to; ++n) {
      if (++trials_ > 16384) return true;
      if (reach(i + 1, left - n * s.length)) return true;
    }
    return false;
  }
  Step steps_[9];
  Wide least_[10] = {}, most_[10] = {}, distance_;
  int n_ = 0, trials_ = 0;
  bool empty_;
};

// Whether the spans of their addresses meet, which mostly settles it (and costs the host little).
inline bool meet(const Operand& x, const Operand& y, int bytes) {
  auto reach = [&](const Operand& o, __int128* from, __int128* to) {
    *from = *to = static_cast<__int128>(reinterpret_cast<uintptr_t>(o.at));
    for (int i = 0; i < o.axes; ++i) {
      const __int128 far = static_cast<__int128>(o.size[i] - 1) * o.stride[i] * bytes;
      *(far < 0 ? from : to) += far;
    }
    *to += bytes;
  };
  __int128 x0, x1, y0, y1;
  reach(x, &x0, &x1);
  reach(y, &y0, &y1);
  return x0 < y1 && y0 < x1;
}

// Whether two elements of one operand stand in the same place: whether steps along its axes, not
// all 0, lead back.  An axis that lies inside the next one's stride settles it for all before.
class Repeating {
 public:
  explicit Repeating(const Operand& x) {
    for (int i = 0; i < x.axes; ++i) {
      if (x.size[i] < 1) empty_ = true;
      if (x.size[i] < 2) continue;
      const Wide stride = x.stride[i] < 0 ? -static_cast<Wide>(x.stride[i]) : x.stride[i];
      int at = n_++;      // the shortest first
      for (; at && stride_[at - 1] > stride; --at) {
        stride_[at] = stride_[at - 1];
        last_[at] = last_[at - 1];
      }
      stride_[at] = stride;
      last_[at] = x.size[i] - 1;
    }
  }
  bool operator()() {
    if (empty_) return false;
    Wide span = 0;      // of the axes below i
    for (int i = 0; i < n_; ++i) {
      if (stride_[i] <= span)
        for (Wide k = 1; k <= last_[i] && k * stride_[i] <= span; ++k) {
          if (++trials_ > 16384 || back(i - 1, span, k * stride_[i])) return true;
        }
      if (stride_[i] == 0) return true;
      span += stride_[i] * last_[i];
    }
    return false;
  }

 private:
  using Wide = __int128;
  // whether steps along axes 0 .. i, which reach `span` to either side, make up `left`
  bool back(int i, Wide span, Wide left) {
    if (left == 0) return true;
    if (i < 0 || left > span || -left > span) return false;
    const Wide below = span - stride_[i] * last_[i];
    for (Wide k = -last_[i]; k <= last_[i]; ++k) {
      const Wide rest = left - k * stride_[i];
      if (rest > below || -rest > below) continue;
      if (++trials_ > 16384 || back(i - 1, below, rest)) return true;
    }
    return false;
  }
  Wide stride_[4], last_[4];
  int n_ = 0, trials_ = 0;
  bool empty_ = false;
};

// Refuses an output whose own elements share memory.
inline int once(const char* what, const Operand& out) {
  if (!Repeating(out)()) return 0;
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: %s is written, but its elements share memory", what,
                out.name);
  return tg_fail(-1, msg);
}

// Refuses an output that shares memory with another operand.
inline int apart(const char* what, const Operand& out, const Operand& x, int bytes) {
  if (!meet(out, x, bytes) || !Sharing(out, x, bytes)()) return 0;
  char msg[256];
  std::snprintf(msg, sizeof(msg), "%s: %s overlaps %s", what, out.name, x.name);
  return tg_fail(-1, msg);
}

}  // namespace tg
