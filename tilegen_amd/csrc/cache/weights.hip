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
  int parts, part_rows;   // wide: a sequence's rows are cut into parts of so many
  float scale, decay;     // scale * log2 e
  Div by_group, by_heads, by_splits, by_parts;
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

// A workgroup takes `chunk` keys of a sequence's for one kv head, each wave every fourth tile.
template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves) void weigh_narrow(Weights a) {
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, quad = lane >> 4;
  const int unit = a.by_heads(blockIdx.x), kv_head = blockIdx.x - unit * a.kv_heads;
  const int b = a.by_splits(unit), split = unit - b * a.splits;
  const Own s = own_of(a.table, b);
  if (s.count == 0) return;
  const int k1 = split + 1 < a.splits ? min(s.keys, (split + 1) * a.chunk) : s.keys;
  const T* kc = static_cast<const T*>(a.key_cache) + kv_head * a.kc_head;
  const int rows = s.count * a.group;

  for (int key0 = split * a.chunk + 32 * wave; key0 < k1; key0 += 32 * kWaves) {
    s16x8 k[2][KS];
    float* at[2];
    bool bad[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = min(key0 + 16 * t + col, k1 - 1);
      const int nth = a.table.by_page(key), slot = key - nth * a.table.page;
      const i64 page = s.list[nth];
      bad[t] = page < 0 || page >= a.table.pages;
      const T* from = kc + (bad[t] ? 0 : page * a.kc_page + slot * a.kc_slot) + 8 * quad;
      at[t] = a.weights + (bad[t] ? 0 : page * a.w_page + slot * a.w_slot + kv_head * a.w_head);
#pragma unroll
      for (int i = 0; i < KS; ++i)
        k[t][i] = !bad[t] && 32 * i + 8 * quad < a.dim
                      ? __builtin_bit_cast(s16x8, C::load(from + 32 * i))
                      : s16x8(0);
    }
    float sum[2][4] = {};
    // the first token that sees the tile's first key
    const int j0 = max(key0 - s.before, 0);
    for (int row0 = j0 * a.group & ~15; row0 < rows; row0 += 16) {
      const int row = row0 + col;
      const bool live = row < rows;
      const int j = a.by_group(live ? row : rows - 1);
      const int h = kv_head * a.group + (live ? row : rows - 1) - j * a.group;
      const T* from = static_cast<const T*>(a.query) + (s.first + j) * a.q_token + h * a.q_head +
                      8 * quad;
      const float lse = a.lse[(s.first + j) * a.l_token + h * a.l_head];
      const int see = live && lse != -INFINITY ? s.before + j + 1 : 0;
      const float base = lse * kLog2e;
      s16x8 q[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i)
        q[i] = 32 * i + 8 * quad < a.dim ? __builtin_bit_cast(s16x8, C::load(from + 32 * i))
                                         : s16x8(0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 sc = f32x4(0.f);
#pragma unroll
        for (int i = 0; i < KS; ++i) sc = M::mul16(k[t][i], q[i], sc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.scale, -base));
          sum[t][i] += key0 + 16 * t + 4 * quad + i < see ? e : 0.f;
        }
      }
    }
    // lane (quad, col): the key's own lane is (col of its half); sums stand by quads
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float all = sum16(sum[t][i]);
        const float v = __shfl(all, (col >> 2) * 16);
        if ((col & 3) == i) mine = v;
      }
      const int key = key0 + 16 * t + col;
      if (quad == 0 && key < k1 && !bad[t])
        *at[t] = (key < s.before ? a.decay * *at[t] : 0.f) + mine;
    }
  }
}

// Many rows.  A wave keeps KT tiles of 32 keys in registers, a workgroup reads the rows once for its
// four: the next stage of 64 rows is in flight to registers while this one's scores are taken from
// LDS.
template <int DP>
struct Wide {
  static constexpr int KT = DP > 128 ? 1 : 2;             // tiles of a wave
  static constexpr int kKeys = 32 * KT * kWaves;          // of a workgroup
  static constexpr int kRows = 64;                        // of a stage
  static constexpr int kUnits = DP / 8;                   // of 16 bytes of a row
  static constexpr int kRow = DP * 2 + 16;                // bytes of a row in LDS: an odd number of units
  static constexpr int kEach = kRows * kUnits / (64 * kWaves);
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_wide(Weights a) {
  using W = Wide<DP>;
  using M = Matrix<T>;
  using C = Chunk<T>;
  constexpr int KS = DP / 16, KT = W::KT;
  __shared__ __align__(16) char s_rows[2][W::kRows * W::kRow];
  __shared__ float s_base[2][W::kRows];
  __shared__ int s_see[2][W::kRows];
  __shared__ int s_strange[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, half = lane >> 5;
  // the kv heads side by side (each XCD has its own of 8), the parts of the same keys next
  const int unit = a.by_heads(blockIdx.x), kv_head = blockIdx.x - unit * a.kv_heads;
  const int up = a.by_parts(unit), part = unit - up * a.parts;
  const int b = a.by_splits(up), split = up - b * a.splits;
  const Own s = own_of(a.table, b);
  const int first_key = split * W::kKeys;
  if (s.count == 0 || first_key >= s.keys) return;
  const int rows = s.count * a.group;
  const int key_blocks = split + 1 < a.splits ? 1 : (s.keys - first_key + W::kKeys - 1) / W::kKeys;
  const T* q_head = static_cast<const T*>(a.query) + s.first * a.q_token +
                    kv_head * a.group * a.q_head;
  const float* l_head = a.lse + s.first * a.l_token + kv_head * a.group * a.l_head;
  const T* kc = static_cast<const T*>(a.key_cache) + kv_head * a.kc_head;

  // (keys past the bound that sized the launch: the last split takes them in turn, its first part
  // with all rows)
  for (int block = 0; block < key_blocks && (block == 0 || part == 0); ++block) {
    const bool whole = a.parts == 1 || block > 0;
    const int key0 = first_key + block * W::kKeys + wave * 32 * KT;
    // from the first token that sees the first key on
    const int seen_from =
        (max(first_key + block * W::kKeys - s.before, 0) * a.group) & -W::kRows;
    const int row_begin = whole ? seen_from : max(seen_from, part * a.part_rows);
    const int row_end =
        whole || part + 1 == a.parts ? rows : min(rows, (part + 1) * a.part_rows);
    if (!whole && row_begin >= row_end) continue;
    s16x8 k[KT][KS];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = min(key0 + 32 * t + col, s.keys - 1);
      const int nth = a.table.by_page(key);
      const i64 page = s.list[nth];
      const bool bad = page < 0 || page >= a.table.pages;
      const T* from =
          kc + (bad ? 0 : page * a.kc_page + (key - nth * a.table.page) * a.kc_slot) + 8 * half;
#pragma unroll
      for (int i = 0; i < KS; ++i)
        k[t][i] = !bad && 16 * i + 8 * half < a.dim
                      ? __builtin_bit_cast(s16x8, C::load(from + 16 * i))
                      : s16x8(0);
    }
    float sum[KT][16];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[t][i] = 0.f;

    s16x8 next[W::kEach];
    float next_lse = 0.f;
    int next_see = 0;
    auto load = [&](int row0) {
#pragma unroll
      for (int i = 0; i < W::kEach; ++i) {
        const int at = tid + i * 64 * kWaves, r = at / W::kUnits, d = (at - r * W::kUnits) * 8;
        const int row = min(row0 + r, rows - 1), j = a.by_group(row);
        next[i] = d < a.dim ? __builtin_bit_cast(s16x8, C::load(q_head + j * a.q_token +
                                                                (row - j * a.group) * a.q_head + d))
                            : s16x8(0);
      }
      if (wave == 0) {
        const int row = min(row0 + lane, rows - 1), j = a.by_group(row);
        next_lse = l_head[j * a.l_token + (row - j * a.group) * a.l_head];
        next_see = row0 + lane < row_end && next_lse != -INFINITY ? s.before + j + 1 : 0;
      }
    };
    auto put = [&](int to) {
#pragma unroll
      for (int i = 0; i < W::kEach; ++i) {
        const int at = tid + i * 64 * kWaves, r = at / W::kUnits, u = at - r * W::kUnits;
        *reinterpret_cast<s16x8*>(&s_rows[to][r * W::kRow + u * 16]) = next[i];
      }
      if (wave == 0) {
        s_base[to][lane] = next_lse * kLog2e;
        s_see[to][lane] = next_see;
        const int strange = __any(next_see == 0);
        if (lane == 0) s_strange[to] = strange;
      }
    };
    if (row_begin < row_end) {
      load(row_begin);
      put(0);
    }
    __syncthreads();
    int at = 0;
    for (int row0 = row_begin; row0 < row_end; row0 += W::kRows, at ^= 1) {
      const bool more = row0 + W::kRows < row_end;
      if (more) load(row0 + W::kRows);
      // every row of the stage sees every key of the wave's, or some may not
      const bool masked =
          s_strange[at] || s.before + static_cast<int>(a.by_group(row0)) + 1 < key0 + 32 * KT;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const char* from = &s_rows[at][(32 * h + col) * W::kRow + 16 * half];
        s16x8 q[KS];
#pragma unroll
        for (int i = 0; i < KS; ++i) q[i] = *reinterpret_cast<const s16x8*>(from + 32 * i);
        const float base = s_base[at][32 * h + col];
        const int see = s_see[at][32 * h + col];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          f32x16 sc = f32x16(0.f);
#pragma unroll
          for (int i = 0; i < KS; ++i) sc = M::mul32(k[t][i], q[i], sc);
          if (!masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              sum[t][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.scale, -base));
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.scale, -base));
              const int key = key0 + 32 * t + 8 * (i / 4) + 4 * half + i % 4;
              sum[t][i] += key < see ? e : 0.f;
            }
          }
        }
      }
      if (more) put(at ^ 1);
      __syncthreads();
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
          a.part[(static_cast<i64>(unit) * a.kv_heads + kv_head) * W::kKeys + key - first_key] = mine;
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
  const int rows = s.count * a.group;
  const int seen_from = (max(first_key - s.before, 0) * a.group) & -64;
  const int last = min(a.parts - 1, (rows - 1) / a.part_rows);
  float sum = 0.f;
  for (int part = min(seen_from / a.part_rows, a.parts - 1); part <= last; ++part)
    sum += a.part[((static_cast<i64>(unit) * a.parts + part) * a.kv_heads + kv_head) * keys +
                  threadIdx.x];
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
  int64_t groups, bytes;
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
  if (rows > 32) {
    p->keys = a.dim > 128 ? 128 : 256;
    a.splits = static_cast<int>((length + p->keys - 1) / p->keys);
    // Parts of the rows, at least 16 stages each, while there are few workgroups: earlier keys are
    // seen by more rows, so that a round of workgroups with all rows ends with a few long ones.
    const int64_t units = heads * a.splits, stages = (rows + 63) / 64;
    int64_t parts = units ? 2048 / units : 1;
    if (parts > stages / 16) parts = stages / 16;
    if (parts > 1) {
      a.part_rows = static_cast<int>((stages + parts - 1) / parts * 64);
      a.parts = static_cast<int>((rows + a.part_rows - 1) / a.part_rows);
    }
    p->groups = units * a.parts;
    if (a.parts > 1) p->bytes = p->groups * p->keys * 4;
  } else {
    a.chunk = 128;
    a.splits = static_cast<int>((length + a.chunk - 1) / a.chunk);
    p->groups = heads * a.splits;
  }
  a.by_splits = Div(a.splits);
  a.by_parts = Div(a.parts);
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
    e = launch(reinterpret_cast<const void*>(&join_weights), p.groups / a.parts, 256, more, st);
  }
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
