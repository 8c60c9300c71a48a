// The attention weight that each cached key receives (launch_attention_weights).
//
// weight[p] = (p < before ? decay weight[p] : 0) + the sum over the rows (new token x query head
// of the group) that see p of exp(scale q . k[p] - lse[row]).
//
// Scores are computed transposed, S^T = K Q^T, on 16x16x32 matrix instructions: a lane holds one
// query row (lane % 16) and four keys of each half of a tile of 32, so that a row's logarithm is
// one register and a key's sum stays in its lane until all rows are through.
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
  int heads, kv_heads, group, dim, chunk, splits;
  float scale, decay;     // scale * log2 e
  Div by_group, by_heads, by_splits;
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
      const float base = lse * 1.44269504088896340736f;
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

template <typename T>
const void* kernel_of(int dim) {
  if (dim <= 64) return reinterpret_cast<const void*>(&weigh_narrow<T, 64>);
  if (dim <= 96) return reinterpret_cast<const void*>(&weigh_narrow<T, 96>);
  if (dim <= 128) return reinterpret_cast<const void*>(&weigh_narrow<T, 128>);
  return reinterpret_cast<const void*>(&weigh_narrow<T, 256>);
}

struct Plan {
  Weights a;
  int64_t groups, bytes;
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
  a.chunk = 128;
  a.splits = static_cast<int>((length + a.chunk - 1) / a.chunk);
  a.by_splits = Div(a.splits);
  p->groups = heads * a.splits;
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
  void* args[] = {&a};
  const hipError_t e =
      launch(r->dtype == TG_F16 ? kernel_of<_Float16>(a.dim) : kernel_of<__bf16>(a.dim), p.groups,
             64 * kWaves, args, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
