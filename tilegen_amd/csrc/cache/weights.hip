// The attention weight that each cached key receives (launch_attention_weights).
//
// weight[p] = (p < before ? decay weight[p] : 0) + the sum over the rows (new token x query head
// of the group) that see p of exp(scale q . k[p] - lse[row]).
//
// Scores are computed transposed, S^T = K Q^T: a lane holds one query row and several keys, so
// that a row's logarithm is one register and a key's sum stays in its lane until all rows are
// through.  Few rows: 16x16x32 matrix instructions, each wave with keys of its own (narrow).
// Many: 32x32x16, keys in registers, rows through LDS for a workgroup (wide).
#include "../attention/parts.h"
#include "cache.h"

#include <type_traits>

namespace tg {
namespace {

struct Weights {
  const void* query;
  const float* lse;
  const void* key_cache;
  float* weights;
  Table table;
  i64 q_token, q_head, l_token, l_head, kc_page, kc_slot, kc_head, w_page, w_slot, w_head;
  float* part;            // [unit, part, keys of a workgroup]: sums of a part of the rows
  int heads, kv_heads, group, dim, chunk, splits;
  int parts, part_stages; // wide: a sequence's stages of rows are cut into parts of so many,
  int large, last_stages; // the first `large` of them, the others of these
  int stage_rows;         // of 64: whole tokens' where a group fits
  int packed;             // the pieces that there are come first, the others of the launch last
  float scale, decay;     // scale * log2 e
  Div by_group, by_heads, by_splits, by_parts, by_stage, by_sequences;
};

__device__ __forceinline__ float sum16(float v) {
  auto add = [](float x, auto order) {
    const int i = __builtin_bit_cast(int, x);
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, i, decltype(order)::value,
                                                                     0xF, 0xF, true));
  };
  v = add(v, std::integral_constant<int, 0xB1>{});
  v = add(v, std::integral_constant<int, 0x4E>{});
  v = add(v, std::integral_constant<int, 0x141>{});
  return add(v, std::integral_constant<int, 0x140>{});
}

// Few rows.  A wave takes `chunk` keys of a sequence's for one kv head, in tiles of 32; the kv heads
// of the same keys follow one another, a workgroup's waves too, so that what is read together lies
// together (32 sequences of up to 4096 keys, 8 kv heads of 128: 4% faster than with one head's next
// keys in a workgroup's waves).  The next tile's keys and weights are asked for as soon as this
// one's products have taken the registers, their pages a tile earlier.  Memory bounds it: 8 kv heads
// of 131072 keys (268 MB) take 55 us, 4.9 TB/s.
template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves) void weigh_narrow(Weights a) {
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int task = blockIdx.x * kWaves + wave;
  const int unit = a.by_heads(task), kv_head = task - unit * a.kv_heads;
  int b, split;
  Own s;
  if (!a.packed) {
    b = a.by_splits(unit);
    split = unit - b * a.splits;
    if (b >= a.table.sequences) return;
    s = own_of(a.table, b);
  } else {
    // the unit-th piece of those that there are, a lane for each of 64 sequences
    Own own;
    int n, sum, before = 0, b0 = 0;
    uint64_t past;
    for (;; b0 += 64) {
      if (b0 >= a.table.sequences) return;
      own = own_of(a.table, min(b0 + lane, a.table.sequences - 1));
      n = b0 + lane < a.table.sequences && own.count
              ? min((own.keys + a.chunk - 1) / a.chunk, a.splits) : 0;
      sum = before + upto(n);
      past = __ballot(unit < sum);
      if (past) break;
      before = __builtin_amdgcn_readlane(sum, 63);
    }
    const int at = __builtin_ctzll(past);
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
    const i64 list = reinterpret_cast<i64>(own.list);
    b = b0 + at;
    split = unit - of(sum - n);
    s.first = of(own.first);
    s.count = of(own.count);
    s.before = of(own.before);
    s.keys = of(own.keys);
    s.list = reinterpret_cast<const int64_t*>(
        static_cast<i64>(of(static_cast<int>(list >> 32))) << 32 |
        static_cast<uint32_t>(of(static_cast<int>(list))));
  }
  const int k1 = split + 1 < a.splits ? min(s.keys, (split + 1) * a.chunk) : s.keys;
  int key0 = split * a.chunk;
  if (s.count == 0 || key0 >= k1) return;
  const T* kc = static_cast<const T*>(a.key_cache) + kv_head * a.kc_head;
  float* weights = a.weights + kv_head * a.w_head;
  const int rows = s.count * a.group;

  // keys key0 + 16 t + col (past the end: the last one): pages, then keys and what they weighed
  i64 page[2];
  int slot[2];
  auto find = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = min(from + 16 * t + col, k1 - 1), nth = a.table.by_page(key);
      slot[t] = key - nth * a.table.page;
      page[t] = s.list[nth];
    }
  };
  s16x8 k[2][KS];
  float* at[2];
  float old[2];
  auto load = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool bad = page[t] < 0 || page[t] >= a.table.pages;
      const T* x = kc + (bad ? 0 : page[t] * a.kc_page + slot[t] * a.kc_slot);
      at[t] = bad ? nullptr : weights + page[t] * a.w_page + slot[t] * a.w_slot;
#pragma unroll
      for (int i = 0; i < KS; ++i) {    // (elements past the head: any of it, times zero)
        const int d = 32 * i + 8 * quad;
        k[t][i] = __builtin_bit_cast(s16x8, C::load(x + (d < a.dim ? d : 0)));
        if (d >= a.dim) k[t][i] = s16x8(0);
      }
      old[t] = 0.f;
      if (quad == 0 && at[t] && from + 16 * t + col < min(k1, s.before)) old[t] = *at[t];
    }
  };
  s16x8 q[KS];
  int see = 0;
  float base = 0.f;
  auto row_tile = [&](int row0) __attribute__((always_inline)) {
    const int row = min(row0 + col, rows - 1), j = a.by_group(row);
    const int h = kv_head * a.group + row - j * a.group;
    const T* x = static_cast<const T*>(a.query) + (s.first + j) * a.q_token + h * a.q_head;
    const float lse = a.lse[(s.first + j) * a.l_token + h * a.l_head];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int d = 32 * i + 8 * quad;
      q[i] = __builtin_bit_cast(s16x8, C::load(x + (d < a.dim ? d : 0)));
      if (d >= a.dim) q[i] = s16x8(0);
    }
    see = row0 + col < rows && lse != -INFINITY ? s.before + j + 1 : 0;
    base = lse * kLog2e;
  };

  find(key0);
  if (rows <= 16) row_tile(0);
  load(key0);
  find(key0 + 32);
  for (; key0 < k1; key0 += 32) {
    float sum[2][4] = {};
    float* to[2];
    float had[2];
    bool loaded = false;
    auto next = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        to[t] = at[t];
        had[t] = old[t];
      }
      if (key0 + 32 < k1) {
        load(key0 + 32);
        find(key0 + 64);
      }
      loaded = true;
    };
    // from the first token that sees the tile's first key on
    const int from = (max(key0 - s.before, 0) * a.group) & ~15;
    for (int row0 = from; row0 < rows; row0 += 16) {
      if (rows > 16) row_tile(row0);
      f32x4 sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = f32x4(0.f);
#pragma unroll
        for (int i = 0; i < KS; ++i) sc[t] = M::mul16(k[t][i], q[i], sc[t]);
      }
      if (row0 + 16 >= rows) next();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], a.scale, -base));
          sum[t][i] += key0 + 16 * t + 4 * quad + i < see ? e : 0.f;
        }
    }
    if (!loaded) next();
    // over the 16 rows that lanes hold; lane c of the first quad writes key c, whose sum is with quad
    // c / 4
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = __shfl(sum16(sum[t][i]), (col >> 2) * 16);
        if ((col & 3) == i) mine = v;
      }
      const int key = key0 + 16 * t + col;
      if (quad == 0 && to[t] && key < k1)
        *to[t] = (key < s.before ? a.decay * had[t] : 0.f) + mine;
    }
  }
}

// Many rows.  A wave keeps KT tiles of 32 keys in registers, a workgroup reads the rows for its four:
// a stage of up to 64 rows (of heads over 128 32), whole tokens', is taken from LDS while the next
// one comes, straight to LDS (4 prompts of up to 4096 tokens on up to 8192 older keys, 325 GFLOP, took
// 399 us so and 413 through registers).  A tile's exponentials and sums run between the products of
// the next tile: 8 products of 32 cycles beside 16 times (fma, exponential, add) of 4, 8 and 4, which
// by themselves take 256 and 268 cycles of a SIMD and together, from registers alone, 412.  Here a
// tile takes about 570: one sequence of 4096 tokens on 8192 older keys, 32/8 heads of 128, 348 GFLOP,
// 363 us, 958 TFLOP/s (with zeros for operands it took 323 of 376 us: power is part of it).  4
// prompts of up to 4096 tokens take 144 us, 825 TFLOP/s: the start of a workgroup, masked halves and
// the last workgroups' end are the rest.  The same prompts with heads of 64, 80 and 96 take 126 us,
// where exponentials are most of it, and with heads of 256 296 us, 799 TFLOP/s.
constexpr int wide_rows(int dim) { return dim > 128 ? 32 : 64; }

template <int DP>
struct Wide {
  static constexpr int KT = DP > 128 ? 1 : 2;             // tiles of a wave
  static constexpr int kKeys = 32 * KT * kWaves;          // of a workgroup
  static constexpr int kRows = wide_rows(DP);             // of a stage, some of them empty
  static constexpr int kUnits = DP / 8;                   // of 16 bytes of a row
  static constexpr int kEach = kRows * kUnits / (64 * kWaves);    // units that a lane brings
  // Rows come straight to LDS, 16 bytes a lane side by side, so they cannot be padded: a row's units
  // change places instead, and a lane brings the unit that belongs to its place.  8 rows' units of one
  // number then lie in all banks (16 rows' where a row has 256 bytes).
  static __device__ __forceinline__ int place(int row) {
    return DP == 64 ? row >> 1 & 7 : DP == 96 ? row >> 1 & 3 : row & 15;
  }
};

// Where a part begins (the last ends with the rows), and whose a stage is.
__device__ __forceinline__ int part_begin(const Weights& a, int part) {
  return min(part, a.large) * a.part_stages + max(part - a.large, 0) * a.last_stages;
}
__device__ __forceinline__ int part_of(const Weights& a, int stage) {
  const int past = stage - a.large * a.part_stages;
  return min(past < 0 ? stage / a.part_stages : a.large + past / a.last_stages, a.parts - 1);
}

// Splits of a sequence's keys that a part of its rows sees; all, if there are more keys than the bound
// that sized the launch and the part is the one that takes them.
constexpr int kPairs = 1024;      // of parts and sequences
template <int KEYS>
__device__ __forceinline__ int pieces_of(const Weights& a, const Own& s, int part) {
  const int stages = a.by_stage(s.count * a.group + a.stage_rows - 1);
  if (part_begin(a, part) >= stages) return 0;
  if (part == 0 && s.keys > a.splits * KEYS) return a.splits;
  const int end = part + 1 < a.parts ? min(stages, part_begin(a, part + 1)) : stages;
  const int tokens = min(s.count, end * a.by_group(a.stage_rows));
  return min((max(0, min(s.before + tokens, s.keys)) + KEYS - 1) / KEYS, a.splits);
}

// 16 bytes of every lane to LDS at `to` + 16 * lane, without a register between.
__device__ __forceinline__ void units_to_lds(__amdgpu_buffer_rsrc_t memory, uint32_t at, char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(memory, (__attribute__((address_space(3))) void*)to, 16,
                                           at, 0, 0, 0);
}

template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_wide(Weights a) {
  using W = Wide<DP>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 16, KT = W::KT;
  // (two arrays: reads of one need not wait for what comes to the other)
  __shared__ __align__(16) char s_even[W::kRows * 2 * DP], s_odd[W::kRows * 2 * DP];
  __shared__ float s_base[2][W::kRows];
  __shared__ int s_see[2][W::kRows];
  __shared__ int s_strange[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  // the kv heads side by side (each XCD has its own of 8), then those that read the same rows
  const int unit = a.by_heads(blockIdx.x), kv_head = blockIdx.x - unit * a.kv_heads;
  int b, part, split;
  Own s;
  if (!a.packed) {
    const int up = a.by_splits(unit);
    split = unit - up * a.splits;
    b = a.by_parts(up);
    part = up - b * a.parts;
    s = own_of(a.table, b);
  } else {
    // the unit-th piece of those that there are: a part's splits follow one another
    __shared__ int s_sum[kWaves];
    __shared__ struct {
      Own s;
      int b, part, split;
    } s_piece;
    const int pairs = a.parts * a.table.sequences;
    if (tid == 0) s_piece.part = -1;
    int before = 0;
    for (int pair0 = 0; pair0 < pairs && before <= unit; pair0 += 64 * kWaves) {
      const int pair = pair0 + tid, nth = a.by_sequences(pair);
      const Own own = own_of(a.table, pair < pairs ? pair - nth * a.table.sequences : 0);
      const int n = pair < pairs ? pieces_of<W::kKeys>(a, own, nth) : 0;
      int sum = upto(n);
      if (lane == 63) s_sum[wave] = sum;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w == wave) sum += before;
        before += s_sum[w];
      }
      // (before: all so far; sum: those up to this thread's)
      if (unit < sum && unit >= sum - n) {
        s_piece.s = own;
        s_piece.b = pair - nth * a.table.sequences;
        s_piece.part = nth;
        s_piece.split = unit - (sum - n);
      }
      __syncthreads();
    }
    if (s_piece.part < 0) return;
    b = __builtin_amdgcn_readfirstlane(s_piece.b);
    part = __builtin_amdgcn_readfirstlane(s_piece.part);
    split = __builtin_amdgcn_readfirstlane(s_piece.split);
    s = s_piece.s;
  }
  const int first_key = split * W::kKeys;
  if (s.count == 0 || first_key >= s.keys) return;
  const int rows = s.count * a.group;
  const int stages = a.by_stage(rows + a.stage_rows - 1);
  const int key_blocks = split + 1 < a.splits ? 1 : (s.keys - first_key + W::kKeys - 1) / W::kKeys;
  const T* q_head = static_cast<const T*>(a.query) + s.first * a.q_token +
                    kv_head * a.group * a.q_head;
  const float* l_head = a.lse + s.first * a.l_token + kv_head * a.group * a.l_head;
  const T* kc = static_cast<const T*>(a.key_cache) + kv_head * a.kc_head;

  // where this lane's units of a stage stand from its first row, in bytes; past the last of `left`
  // rows the last, past the head its first unit (and zero in the keys)
  auto units_of = [&](int left, uint32_t (&off)[W::kEach]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < W::kEach; ++i) {
      const int at = (i * kWaves + wave) * 64 + lane, nth = at / W::kUnits;
      const int r = min(nth, left - 1), j = a.by_group(r), unit = at % W::kUnits ^ W::place(nth);
      off[i] = static_cast<uint32_t>(2 * (j * a.q_token + (r - j * a.group) * a.q_head +
                                          (unit * 8 < a.dim ? unit * 8 : 0)));
    }
  };
  uint32_t all[W::kEach];
  units_of(a.stage_rows, all);

  // (keys past the bound that sized the launch: the last split takes them in turn, its first part
  // with all rows)
  for (int block = 0; block < key_blocks && (block == 0 || part == 0); ++block) {
    const bool whole = a.parts == 1 || block > 0;
    const int key0 = first_key + block * W::kKeys + wave * 32 * KT;
    // from the first token that sees the first key on
    const int seen_from =
        a.by_stage(max(first_key + block * W::kKeys - s.before, 0) * a.group);
    const int begin = whole ? seen_from : max(seen_from, part_begin(a, part));
    const int end = whole || part + 1 == a.parts ? stages : min(stages, part_begin(a, part + 1));
    if (!whole && begin >= end) continue;
    float next_lse = 0.f;
    int next_see = 0;
    auto load = [&](int stage, auto odd) __attribute__((always_inline)) {
      const int row0 = stage * a.stage_rows, left = min(rows - row0, a.stage_rows);
      const T* from = q_head + static_cast<i64>(a.by_group(row0)) * a.q_token;
      const auto memory = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(from), 0, 0x7FFFFFFF,
                                                            0x00027000);
      char* to = (decltype(odd)::value ? s_odd : s_even) + wave * 1024;
      if (wave == 0) {
        const int row = min(row0 + lane, rows - 1), j = a.by_group(row);
        next_lse = l_head[j * a.l_token + (row - j * a.group) * a.l_head];
        next_see = lane < left ? s.before + j + 1 : INT32_MIN;
      }
      uint32_t off[W::kEach];
#pragma unroll
      for (int i = 0; i < W::kEach; ++i) off[i] = all[i];
      if (left < a.stage_rows) units_of(left, off);
#pragma unroll
      for (int i = 0; i < W::kEach; ++i)
        units_to_lds(memory, off[i], to + i * kWaves * 1024);
    };
    auto put = [&](int to) __attribute__((always_inline)) {
      if (wave == 0) {
        const bool live = next_see != INT32_MIN;
        if (lane < W::kRows) {
          s_base[to][lane] = live ? next_lse * kLog2e : INFINITY;
          s_see[to][lane] = live && next_lse != -INFINITY ? next_see : 0;
        }
        const int strange = __any(live && !(fabsf(next_lse) < INFINITY));
        if (lane == 0) s_strange[to] = strange;
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // what this wave brings is there
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> uneven;

    s16x8 k[KT][KS];
    const T* k_at[KT];
    bool bad[KT];
    i64 page[KT];
    int slot[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = min(key0 + 32 * t + col, s.keys - 1), nth = a.table.by_page(key);
      page[t] = s.list[nth];
      slot[t] = key - nth * a.table.page;
    }
    if (begin < end) load(begin, even);     // (on its way beside the keys, behind their pages)
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      bad[t] = page[t] < 0 || page[t] >= a.table.pages;
      k_at[t] = kc + (bad[t] ? 0 : page[t] * a.kc_page + slot[t] * a.kc_slot);
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int i = 0; i < KS; ++i) {    // (elements past the head: any of it, zero below)
        const int d = 16 * i + 8 * half;
        k[t][i] = __builtin_bit_cast(s16x8, C::load(k_at[t] + (d < a.dim ? d : 0)));
      }
    }
    bool odd = false;     // an infinity or NaN among the keys: rows that are 0 would be NaN
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
        if (bad[t] || 16 * i + 8 * half >= a.dim) k[t][i] = s16x8(0);
      f32x16 zero = f32x16(0.f);
#pragma unroll
      for (int i = 0; i < KS; ++i) zero = M::mul32(k[t][i], s16x8(0), zero);
#pragma unroll
      for (int e = 0; e < 16; ++e) odd |= zero[e] != 0.f;
    }
    odd = __any(odd);
    float sum[KT][16];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[t][i] = 0.f;

    // q: rows 32 h .. of a stage; before: the scores of the tile before, which are added up between
    // the products of this one; see: of the lane's keys, counted from its first
    s16x8 q[KS];
    float base = 0.f, base_before = 0.f;
    int see = 0;
    f32x16 before = f32x16(-INFINITY);
    int in_row = (half ^ W::place(col)) * 16;     // (the same in both halves of 32 rows)
    auto fetch = [&](auto odd, int h, int i) __attribute__((always_inline)) {
      q[i] = *reinterpret_cast<const s16x8*>(&(decltype(odd)::value ? s_odd : s_even)[
          (32 * h + col) * 2 * DP + (2 * i * 16 ^ in_row)]);
    };
    auto fetch_row = [&](auto odd, int h) __attribute__((always_inline)) {
      base = s_base[odd][32 * h + col];
      see = s_see[odd][32 * h + col] - key0 - 4 * half;
    };
    // TILE's products; then, in the last tile of these rows, the rows 32 h of a buffer are read
    auto step = [&](auto tile, bool masked, auto at, int h) __attribute__((always_inline)) {
      constexpr int TILE = decltype(tile)::value, LAST = TILE == KT - 1;
      constexpr int BEFORE = TILE ? TILE - 1 : KT - 1;
      f32x16 sc;
      if (masked) {     // scores start from -inf where a row does not see a key
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sc[e] = 32 * TILE + 8 * (e / 4) + e % 4 < see ? 0.f : -INFINITY;
        sc = M::mul32(k[TILE][0], q[0], sc);
      } else {
        sc = M::mul32(k[TILE][0], q[0], f32x16(0.f));
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if (i) sc = M::mul32(k[TILE][i], q[i], sc);
        if (LAST) fetch(at, h, i);
#pragma unroll
        for (int e = 16 * i / KS; e < 16 * (i + 1) / KS; ++e)
          sum[BEFORE][e] +=
              __builtin_amdgcn_exp2f(__builtin_fmaf(before[e], a.scale, -base_before));
        if (LAST) __builtin_amdgcn_sched_barrier(0);    // (the reads would all come behind the products)
      }
      // (the sums stay here: they would be taken behind all products otherwise)
#pragma unroll
      for (int e = 0; e < 16; ++e) asm volatile("" : "+v"(sum[BEFORE][e]));
      before = sc;
      base_before = base;
      if (LAST) fetch_row(at, h);
    };
    auto rows32 = [&](bool masked, auto at, int h) __attribute__((always_inline)) {
      if (DP > 128) asm volatile("" : "+v"(in_row));    // (16 addresses would not fit beside the rest)
      step(std::integral_constant<int, 0>{}, masked, at, h);
      if constexpr (KT > 1) step(std::integral_constant<int, KT - 1>{}, masked, at, h);
    };

    bool strange = false;
    // the other buffer's rows are there, this one's are in registers and the next go over them
    auto turn = [&](int stage, auto at, int other) __attribute__((always_inline)) {
      if (stage + 1 < end) put(other);
      __syncthreads();
      if (stage + 2 < end) load(stage + 2, at);
    };
    // the rest of a stage's rows, then the first of the next one's
    auto stage_of = [&](int stage, auto at, auto other) __attribute__((always_inline)) {
      strange |= s_strange[at] != 0;
      const int token = a.by_group(stage * a.stage_rows);
      const bool masked = __builtin_amdgcn_readfirstlane(s.before + token + 1 < key0 + 32 * KT);
      if constexpr (W::kRows == 64) rows32(masked, at, 1);
      turn(stage, at, other);
      rows32(masked, other, 0);
    };
    if (begin < end) {
      put(0);
      if (begin + 1 < end) load(begin + 1, uneven);
      __syncthreads();
      // (a wave without a key, or whose keys come later than the workgroup's first, waits for them)
      const int from = key0 < s.keys ? a.by_stage(max(key0 - s.before, 0) * a.group) - begin : end;
      const int mine = begin + (max(__builtin_amdgcn_readfirstlane(from), 0) + (key0 >= s.keys) & ~1);
      int stage = begin;
#pragma unroll 1
      for (; stage < mine && stage < end; stage += 2) {
        turn(stage, even, 1);
        if (stage + 1 < end) turn(stage + 1, uneven, 0);
      }
      if (stage < end) {
#pragma unroll
        for (int i = 0; i < KS; ++i) fetch(even, 0, i);
        fetch_row(even, 0);
      }
#pragma unroll 1
      for (; stage < end; stage += 2) {
        stage_of(stage, even, uneven);
        if (stage + 1 < end) stage_of(stage + 1, uneven, even);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sum[KT - 1][e] += __builtin_amdgcn_exp2f(__builtin_fmaf(before[e], a.scale, -base_before));
    }
    // (a finite key that is hidden from a row: -inf and a score past 32 bits are NaN; sums are not
    // negative, so one of all is NaN where one of them is)
    float all_sums = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) all_sums += sum[t][e];
    strange |= all_sums != all_sums;
    if (__syncthreads_or(odd || strange)) {
      // infinities or NaN among the keys, the logarithms or the sums: once more, adding what is seen
      // alone
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[t][e] = 0.f;
#pragma unroll 1
      for (int stage = begin; stage < end; ++stage) {
        load(stage, even);
        put(0);
        __syncthreads();
#pragma unroll 1
        for (int h = 0; h < W::kRows / 32; ++h) {
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            fetch(even, h, i);
            if (16 * i + 8 * half >= a.dim) q[i] = s16x8(0);
          }
          fetch_row(even, h);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            f32x16 sc = f32x16(0.f);
#pragma unroll
            for (int i = 0; i < KS; ++i) sc = M::mul32(k[t][i], q[i], sc);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], a.scale, -base));
              sum[t][e] += 32 * t + 8 * (e / 4) + e % 4 < see ? x : 0.f;
            }
          }
        }
        __syncthreads();
      }
    }

    // over the 32 rows that lanes hold; lane (half, c) of 16 has key 8 (c / 4) + 4 half + c % 4
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const Both all = quarters(sum16(sum[t][i]));
        if ((lane & 15) == i) mine = all.a + all.b;
      }
      const int c = lane & 15, key = key0 + 32 * t + 8 * (c / 4) + 4 * half + c % 4;
      if (!(lane & 16) && key < s.keys) {
        if (!whole) {
          a.part[((static_cast<i64>(b * a.parts + part) * a.splits + split) * a.kv_heads + kv_head) *
                     W::kKeys + key - first_key] = mine;
        } else {
          const int nth = a.table.by_page(key);
          const i64 page = s.list[nth];
          if (page >= 0 && page < a.table.pages) {
            float* to = a.weights + page * a.w_page + (key - nth * a.table.page) * a.w_slot +
                        kv_head * a.w_head;
            *to = (key < s.before ? a.decay * *to : 0.f) + mine;
          }
        }
      }
    }
    __syncthreads();
  }
}

// The parts of the rows joined, in order; one workgroup for the keys of one, a thread a key.
__global__ __launch_bounds__(256) void join_weights(Weights a, int keys) {
  const int unit = a.by_heads(blockIdx.x), kv_head = blockIdx.x - unit * a.kv_heads;
  const int b = a.by_splits(unit), split = unit - b * a.splits;
  const Own s = own_of(a.table, b);
  const int first_key = split * keys, key = first_key + threadIdx.x;
  if (s.count == 0 || static_cast<int>(threadIdx.x) >= keys || key >= s.keys) return;
  const int stages = a.by_stage(s.count * a.group + a.stage_rows - 1);
  const int seen_from = a.by_stage(max(first_key - s.before, 0) * a.group);
  const int last = part_of(a, stages - 1);
  float sum = 0.f;
  for (int part = part_of(a, seen_from); part <= last; ++part)
    sum += a.part[((static_cast<i64>(b * a.parts + part) * a.splits + split) * a.kv_heads + kv_head) *
                      keys + threadIdx.x];
  const int nth = a.table.by_page(key);
  const i64 page = s.list[nth];
  if (page < 0 || page >= a.table.pages) return;
  float* to =
      a.weights + page * a.w_page + (key - nth * a.table.page) * a.w_slot + kv_head * a.w_head;
  *to = (key < s.before ? a.decay * *to : 0.f) + sum;
}

template <typename T>
const void* wide_of(int dim) {
  if (dim <= 64) return reinterpret_cast<const void*>(&weigh_wide<T, 64>);
  if (dim <= 96) return reinterpret_cast<const void*>(&weigh_wide<T, 96>);
  if (dim <= 128) return reinterpret_cast<const void*>(&weigh_wide<T, 128>);
  return reinterpret_cast<const void*>(&weigh_wide<T, 256>);
}

template <typename T>
const void* narrow_of(int dim) {
  if (dim <= 64) return reinterpret_cast<const void*>(&weigh_narrow<T, 64>);
  if (dim <= 96) return reinterpret_cast<const void*>(&weigh_narrow<T, 96>);
  if (dim <= 128) return reinterpret_cast<const void*>(&weigh_narrow<T, 128>);
  return reinterpret_cast<const void*>(&weigh_narrow<T, 256>);
}

struct Plan {
  Weights a;
  int64_t groups, pieces, bytes;
  int keys;     // of a wide workgroup; 0: narrow
};

int plan(const tg_attention_weights* r, Plan* p) {
  const char* what = "launch_attention_weights";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (r->dtype != TG_BF16 && r->dtype != TG_F16)
    return refuse(-1, what, "dtype must be bfloat16 or float16", r->dtype);
  if (r->dim < 8 || r->dim > 256 || r->dim % 8)
    return refuse(-1, what, "dim must be a multiple of 8 up to 256", r->dim);
  if (const int rc =
          check_table(what, r->sequences, r->pages, r->page, r->n_indices, r->max_length))
    return rc;
  if (r->tokens < 0 || r->max_query < 0) return refuse(-1, what, "negative size", r->tokens);
  if (r->kv_heads < 1 || r->heads < r->kv_heads || r->heads % r->kv_heads)
    return refuse(-1, what, "heads must be a multiple of kv_heads", r->heads);
  if (!(r->scale > 0) || !(r->scale < 1e30) || static_cast<float>(r->scale) == 0.f)
    return refuse(-1, what, "scale must be positive and finite", 0);
  if (!(r->decay >= 0) || !(r->decay < 1e30))
    return refuse(-1, what, "decay must be at least 0 and finite", 0);
  if (r->tokens > 0x1000000 || r->heads > 0x10000 || r->tokens * r->heads > 4 * kMostGroups)
    return refuse(-2, what, "2^26 rows", r->tokens);
  if (!r->query_indptr && r->tokens > r->sequences)
    return refuse(-1, what, "more tokens than sequences without query_indptr", r->tokens);
  const int64_t strides[] = {r->kc_page, r->kc_slot, r->kc_head, r->w_page,
                             r->w_slot,  r->w_head,  r->query_token, r->query_head,
                             r->lse_token, r->lse_head};
  if (const int rc = check_strides(what, strides, 10)) return rc;
  *p = Plan{};
  Weights& a = p->a;
  a.query = r->query;
  a.lse = r->lse;
  a.key_cache = r->key_cache;
  a.weights = r->weights;
  a.table.indptr = r->indptr;
  a.table.indices = r->indices;
  a.table.lengths = r->lengths;
  a.table.ends = r->query_indptr;
  a.table.pages = r->pages;
  a.table.n_indices = r->n_indices;
  a.table.tokens = static_cast<int>(r->tokens);
  // without query_indptr sequence b is token b: those past the tokens have none
  a.table.sequences = static_cast<int>(r->query_indptr ? r->sequences : r->tokens);
  a.table.page = static_cast<int>(r->page);
  a.table.by_page = Div(a.table.page);
  a.q_token = r->query_token;
  a.q_head = r->query_head;
  a.l_token = r->lse_token;
  a.l_head = r->lse_head;
  a.kc_page = r->kc_page;
  a.kc_slot = r->kc_slot;
  a.kc_head = r->kc_head;
  a.w_page = r->w_page;
  a.w_slot = r->w_slot;
  a.w_head = r->w_head;
  a.heads = static_cast<int>(r->heads);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int>(r->dim);
  a.scale = static_cast<float>(r->scale * 1.4426950408889634);
  a.decay = static_cast<float>(r->decay);
  a.by_group = Div(a.group);
  a.by_heads = Div(a.kv_heads);
  const int64_t length = r->max_length > 0 ? r->max_length : 1;
  const int64_t heads = static_cast<int64_t>(a.table.sequences) * a.kv_heads;
  const int64_t bound = r->max_query < r->tokens ? r->max_query : r->tokens;
  const int64_t rows = (r->query_indptr && bound > 0 ? bound : 1) * a.group;   // of a sequence
  a.parts = 1;
  // Wide for many rows, or not so few with much work for all (whole tokens in a stage, within 32 bits
  // of its first).  Rows are the most that a sequence has, spread evenly down to one token's.  32
  // sequences of up to 2048 keys, 8 kv heads of 128: 64 rows 29 us narrow, 33 wide;
  // 128 rows 40 and 36; 512 rows 108 and 56.  8 of up to 1000 keys: 256 rows 19 and 14, 512 rows 32
  // and 18.  One of 16384 keys, 4 kv heads: 64 rows 10 and 12, 256 rows 21 and 16.  4 of up to 700
  // keys, 4 kv heads of 64: 256 rows 9.6 and 13.0, 512 rows 15.5 and 15.9, 1024 rows 27 and 16.  2 of
  // up to 1500, 16 kv heads of 128: 128 rows 9.7 and 10.7.
  const int64_t room = wide_rows(a.dim), tokens = room / a.group;
  auto within = [](int64_t steps, int64_t stride) {
    return steps == 0 || (stride >= 0 && stride <= (int64_t(1) << 28) / steps);
  };
  const bool many = rows > 512 || (rows >= 128 && rows * heads >= (1 << 22) / length);
  // (what goes straight to LDS starts at a multiple of 4 bytes)
  const bool fours = reinterpret_cast<uintptr_t>(r->query) % 4 == 0 && r->query_token % 2 == 0 &&
                     r->query_head % 2 == 0;
  if (many && tokens > 0 && fours && within(tokens - 1, r->query_token) &&
      within(a.group - 1, r->query_head)) {
    p->keys = a.dim > 128 ? 128 : 256;
    a.splits = static_cast<int>((length + p->keys - 1) / p->keys);
    a.stage_rows = static_cast<int>(tokens * a.group);
    a.by_stage = Div(a.stage_rows);
    // Parts of the rows, of 16 stages at least: earlier keys are seen by more rows, so that a round of
    // workgroups with all rows ends with a few long ones.  Of 4 stages while two workgroups a compute
    // unit are not there yet: 1 sequence of 2048 keys, 8 kv heads of 128, 2048 rows 35 us by 16 and
    // 22 by 4; of 512 keys of 64, 2048 rows 31 and 16; with work for all, by 8, 188 instead of 165,
    // since a workgroup spends 9 us on lookups and keys before its first product.
    const int64_t units = heads * a.splits, stages = (rows + a.stage_rows - 1) / a.stage_rows;
    int64_t parts = units ? 4096 / units : 1;
    const int64_t few = units ? 512 / units : 1;
    const int64_t fine = few < stages / 4 ? few : stages / 4;
    if (parts > stages / 16) parts = stages / 16 > fine ? stages / 16 : fine;
    a.part_stages = a.last_stages = static_cast<int>(stages);
    a.large = 1;
    if (parts > 1) {
      a.part_stages = a.last_stages = static_cast<int>((stages + parts - 1) / parts);
      a.parts = static_cast<int>((stages + a.part_stages - 1) / a.part_stages);
      a.large = a.parts;
      // The last quarter in halves where there are some rounds of workgroups: what starts last ends
      // sooner (4 prompts of up to 4096 tokens 144 us, 150 in equal parts, on up to 8192 older keys 355
      // and 399; one of 4096 on 8192 363 and 357).
      if (units * a.parts > 1024 && a.part_stages >= 16) {
        a.large = a.parts * 3 / 4;
        a.last_stages = (a.part_stages + 1) / 2;
        const int rest = static_cast<int>(stages) - a.large * a.part_stages;
        a.parts = a.large + (rest + a.last_stages - 1) / a.last_stages;
      }
    }
    p->groups = p->pieces = units * a.parts;
    if (a.parts > 1) p->bytes = p->pieces * p->keys * 4;
    // Which pieces there are is for the lengths to say, and costs every workgroup a look at all of them:
    // 158 us without, 149 with for 4 prompts of up to 4096 tokens, 26.1 and 22.1 for 4 of up to 1024
    // tokens with 8 heads of their own, 27.5 and 30.6 for 1 of 1024 (512 pieces).
    const int64_t pairs = static_cast<int64_t>(a.parts) * a.table.sequences;
    if (p->pieces > (a.table.sequences > 1 ? 256 : 512) && pairs <= kPairs) {
      a.packed = 1;
      // all the tokens' stages, and a part of each sequence's that is not whole
      const int64_t some = (r->tokens / tokens + a.table.sequences) / a.last_stages + a.table.sequences;
      if (some < pairs) p->groups = some * a.splits * a.kv_heads;
    }
  } else {
    // Two tiles a wave where there are many: one sequence of 131072 keys, 8 kv heads 55.2 us, 58.2
    // by one; 32 of 2048 19.4 and 18.0.
    const int64_t tiles = (length + 31) / 32;
    a.chunk = heads * tiles >= 32768 ? 64 : 32;
    a.splits = static_cast<int>((length + a.chunk - 1) / a.chunk);
    p->groups = (heads * a.splits + kWaves - 1) / kWaves;
    // Waves look for the pieces that there are, by 64 sequences: 32 of up to 4096 keys, 8 kv heads of
    // 128, 31.8 us, 33.3 without; with one kv head 64 of them 11.6 and 15.5; 128 of 2048 60 and 68; 256
    // 129 and 132; 512 of 1024 keys, 4 kv heads of 64, 54 and 50.
    a.packed = a.table.sequences > 1 && a.table.sequences <= 256;
  }
  a.by_splits = Div(a.splits);
  a.by_parts = Div(a.parts);
  a.by_sequences = Div(a.table.sequences > 0 ? a.table.sequences : 1);
  if (p->groups > kMostGroups) return refuse(-2, what, "2^24 workgroups or more", p->groups);
  return 0;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int64_t attention_weights_workspace(
    const tg_attention_weights* r) {
  Plan p;
  if (const int rc = plan(r, &p)) return rc < 0 ? rc : -1;
  return p.bytes;
}

extern "C" __attribute__((visibility("default"))) int launch_attention_weights(
    const tg_attention_weights* r, void* stream) {
  const char* what = "launch_attention_weights";
  Plan p;
  if (const int rc = plan(r, &p)) return rc;
  Weights& a = p.a;
  if (p.groups == 0 || a.table.tokens == 0 || a.table.pages == 0 || a.table.n_indices == 0)
    return 0;
  const Operand query = {"query", r->query, 3, {r->tokens, r->heads, r->dim},
                         {r->query_token, r->query_head, 1}};
  const Operand lse = {"lse", r->lse, 2, {r->tokens, r->heads}, {r->lse_token, r->lse_head}};
  const Operand kc = {"key_cache", r->key_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->kc_page, r->kc_slot, r->kc_head, 1}};
  const Operand w = {"weights", r->weights, 3, {r->pages, r->page, r->kv_heads},
                     {r->w_page, r->w_slot, r->w_head}};
  if (const int rc = once(what, w)) return rc;
  if (const int rc = apart(what, w, lse, 4)) return rc;
  for (const Operand* x : {&query, &kc})
    if (const int rc = apart(what, in_halves(w), *x, 2)) return rc;
  if (!r->query || !r->lse || !r->key_cache || !r->weights || !r->indptr || !r->indices ||
      !r->lengths)
    return refuse(-1, what, "null array", r->tokens);
  if (r->workspace_bytes < p.bytes || (p.bytes && !r->workspace))
    return refuse(-1, what, "the workspace is too small; bytes needed", p.bytes);
  if (reinterpret_cast<uintptr_t>(r->workspace) % 16)
    return refuse(-1, what, "the workspace is not 16-byte aligned", 0);
  a.part = static_cast<float*>(r->workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool half = r->dtype == TG_F16;
  const void* k = p.keys ? half ? wide_of<_Float16>(a.dim) : wide_of<__bf16>(a.dim)
                         : half ? narrow_of<_Float16>(a.dim) : narrow_of<__bf16>(a.dim);
  void* args[] = {&a};
  hipError_t e = launch(k, p.groups, 64 * kWaves, args, st);
  if (e == hipSuccess && a.parts > 1) {
    void* more[] = {&a, &p.keys};
    e = launch(reinterpret_cast<const void*>(&join_weights), p.pieces / a.parts, 256, more, st);
  }
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
