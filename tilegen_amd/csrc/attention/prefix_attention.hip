// launch_prefix_attention: how a call is split into parts, and the kernel that joins them.
#include "prefix_attention.h"

namespace tg {
namespace {

// Joins the parts of each row: M = max m_s, then sum 2^(m_s - M) O_s over sum 2^(m_s - M) l_s.
// A lane holds four elements of the head; where a head takes 16 or 32 lanes the others read
// other parts at the same time (LANES: lanes of one part), and WAVES waves share a row where it
// has many.  Memory bounds it, so the weights come first and the parts' loads wait for nothing:
// 16384 rows of 128 in 7 parts (38 MB by then in the caches) take 11.4 us, 1024 rows in some 17
// take 6.0, most of it latency.
template <typename T, int LANES, int WAVES>
__global__ __launch_bounds__(256) void join_parts(Attention a) {
  constexpr int kAtOnce = WAVES * 64 / LANES;     // parts
  __shared__ float4 s_sum[WAVES == 1 ? 1 : 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const i64 rows = static_cast<i64>(a.tokens) * a.heads;
  const i64 row = static_cast<i64>(blockIdx.x) * (4 / WAVES) + (WAVES == 1 ? wave : 0);
  if (row >= rows) return;
  const int t = static_cast<int>(row / a.heads);
  const int h = static_cast<int>(row - static_cast<i64>(t) * a.heads);
  const int b = a.ends ? sequence_of(a.ends, a.sequences, t) : t;
  int parts = b < a.sequences ? a.prefix_splits : 0;
  if (b < a.sequences && a.own_splits) {
    const Sequence s = sequence(a, b);
    parts += own_parts(a, seen(s, t - s.first));
  }
  const float2* ml = a.part_ml + row;
  float top = -INFINITY;
  for (int s = lane; s < parts; s += 64) top = fmaxf(top, ml[s * rows].x);
#pragma unroll
  for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f;
  for (int s = lane; s < parts; s += 64) {
    const float2 v = ml[s * rows];
    total += v.y * exp2f(v.x - base);
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) total += __shfl_xor(total, x);
  const int d = (lane % LANES) * 4;
  const int first = WAVES == 1 ? lane / LANES : threadIdx.x / LANES;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (d < a.dim) {
    const float* from = a.part + row * a.dim + d;
    const i64 stride = rows * a.dim;
    for (int s0 = first; s0 < parts; s0 += 4 * kAtOnce) {
      float f[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + i * kAtOnce;
        f[i] = 0.f;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < parts) {
          f[i] = exp2f(ml[s * rows].x - base);
          v[i] = *reinterpret_cast<const float4*>(from + s * stride);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[0] += v[i].x * f[i];
        sum[1] += v[i].y * f[i];
        sum[2] += v[i].z * f[i];
        sum[3] += v[i].w * f[i];
      }
    }
  }
  for (int x = LANES; x < 64; x <<= 1)
    for (int i = 0; i < 4; ++i) sum[i] += __shfl_xor(sum[i], x);
  if (WAVES > 1) {
    s_sum[threadIdx.x] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 v = s_sum[64 * w + lane];
      sum[0] += v.x;
      sum[1] += v.y;
      sum[2] += v.z;
      sum[3] += v.w;
    }
  }
  if (lane < LANES && d < a.dim) {
    T* out = static_cast<T*>(a.out) + t * a.o_token + h * a.o_head + d;
    const float f = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = static_cast<T>(total == 0.f ? 0.f : sum[i] * f);
  }
  if (lane == 0 && a.lse) a.lse[row] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
}

int compute_units() {
  static thread_local int cus[64] = {};
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 256;
  if (!cus[device]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess ||
        n < 1)
      n = 256;
    cus[device] = n;
  }
  return cus[device];
}

struct Plan {
  Attention a;
  int prefix_rows, own_rows;    // of one workgroup: narrow 16, wide 128
  int64_t bytes;
  bool whole;                   // one launch, without parts
};

constexpr int64_t kWholeElements = 45056;
constexpr int64_t kMostWorkgroups = 0xFFFFFF;   // of 256 threads: HIP launches under 2^32 threads

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

int check(const tg_prefix_attention* r) {
  const char* what = "launch_prefix_attention";
  if (!r) return refuse(-1, what, "null arguments", 0);
  if (r->dtype != TG_BF16 && r->dtype != TG_F16)
    return refuse(-1, what, "dtype must be bfloat16 or float16", r->dtype);
  if (r->dim < 8 || r->dim > 256 || r->dim % 8)
    return refuse(-1, what, "dim must be a multiple of 8 up to 256", r->dim);
  if (r->tokens < 0 || r->sequences < 0 || r->pages < 0 || r->n_prefix < 0 || r->n_indices < 0 ||
      r->prefix_length < 0 || r->max_query < 0 || r->max_length < 0)
    return refuse(-1, what, "negative size", 0);
  if (r->kv_heads < 1 || r->heads < r->kv_heads || r->heads % r->kv_heads)
    return refuse(-1, what, "heads must be a multiple of kv_heads", r->heads);
  if (r->page < 1 || r->page > INT32_MAX)
    return refuse(-1, what, "page must be 1 to 2^31 - 1", r->page);
  // (in 32 bits: 0 times the -inf of a hidden score would be NaN)
  if (!(r->scale > 0) || !(r->scale < 1e30) || static_cast<float>(r->scale) == 0.f)
    return refuse(-1, what, "scale must be positive and finite", 0);
  if (r->prefix_length > INT32_MAX / 2 || r->max_length > INT32_MAX / 2)
    return refuse(-2, what, "more than 2^30 keys", r->prefix_length);
  if (r->pages > INT32_MAX) return refuse(-2, what, "more than 2^31 pages", r->pages);
  if (r->n_prefix < (r->prefix_length + r->page - 1) / r->page)
    return refuse(-1, what, "prefix_length is past the prefix's pages", r->prefix_length);
  if (r->tokens > 0x1000000 || r->sequences > 0x1000000 || r->heads > 0x10000 ||
      r->tokens * r->heads > 4 * kMostWorkgroups)    // join_parts: 4 rows each
    return refuse(-2, what, "2^26 rows or more than 2^24 sequences", r->tokens);
  if (!r->query_indptr && r->tokens > r->sequences)
    return refuse(-1, what, "more tokens than sequences without query_indptr", r->tokens);
  return 0;
}

int plan(const tg_prefix_attention* r, Plan* p) {
  const char* what = "launch_prefix_attention";
  if (const int rc = check(r)) return rc;
  Attention& a = p->a;
  a = Attention{};
  a.q = r->query;
  a.k = r->key_cache;
  a.v = r->value_cache;
  a.prefix = r->prefix;
  a.indptr = r->indptr;
  a.indices = r->indices;
  a.lengths = r->lengths;
  a.ends = r->query_indptr;
  a.out = r->out;
  a.lse = r->lse;
  a.q_token = r->query_token;
  a.q_head = r->query_head;
  a.o_token = r->out_token;
  a.o_head = r->out_head;
  a.kc_page = r->kc_page;
  a.kc_slot = r->kc_slot;
  a.kc_head = r->kc_head;
  a.vc_page = r->vc_page;
  a.vc_slot = r->vc_slot;
  a.vc_head = r->vc_head;
  a.pages = r->pages;
  a.n_indices = r->n_indices;
  a.tokens = static_cast<int>(r->tokens);
  // without query_indptr sequence b is token b: those past the tokens have none
  a.sequences = static_cast<int>(r->query_indptr ? r->sequences : r->tokens);
  a.heads = static_cast<int>(r->heads);
  a.kv_heads = static_cast<int>(r->kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int>(r->dim);
  a.page = static_cast<int>(r->page);
  a.prefix_length = r->pages ? static_cast<int>(r->prefix_length) : 0;
  a.scale = static_cast<float>(r->scale * 1.4426950408889634);
  a.by_group = Div(a.group);
  a.by_page = Div(a.page);
  // pages of whole groups of 8 keys, keys and values with the same strides, and a group's rows
  // within 32 bits of its first
  a.even = a.page % 8 == 0 && a.kc_page == a.vc_page && a.kc_slot == a.vc_slot &&
           a.kc_page >= 0 && a.kc_slot >= 0 && a.kc_slot < (1 << 24);
  p->bytes = 0;
  p->whole = false;
  if (a.tokens == 0) return 0;
  const int64_t cus = compute_units();
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.group;
  const int64_t bound = r->max_query < a.tokens ? r->max_query : a.tokens;
  const int64_t max_query = r->query_indptr && bound > 0 ? bound : 1;
  const int64_t each = max_query * a.group;    // rows of a sequence's own pages, for one kv head
  const int64_t length = r->max_length > 0 ? r->max_length : 1;
  // workgroups that the chip holds at once
  const int64_t room = a.dim > 128 ? cus : 2 * cus;
  const int64_t heads = static_cast<int64_t>(a.sequences) * a.kv_heads;
  const int64_t tiles16 = (each + 15) / 16;
  // Few keys and no more workgroups than run at once: one launch that reads the prefix for each
  // 16 rows.  A call in parts takes 14.5 us up to some thousand keys (two launches); a whole
  // one 10.6 us with few, 10.8 with 360 keys of 64 elements and 15.1 with 660, 12.4 with 360 of
  // 128 and 18.8 with 660.
  if (heads && (a.prefix_length + r->max_length) * a.dim <= kWholeElements &&
      heads * tiles16 <= room) {
    a.own_tiles = static_cast<int>(tiles16);
    p->whole = true;
    return 0;
  }
  // A sequence's own pages: narrow workgroups read them again for every 16 rows, wide ones
  // once for 128 but with long turns.  4 sequences of 8 to 16 rows run as fast either way; 24 rows
  // of 3 sequences, 1500 keys: 14.5 us narrow, 20.5 wide; 28 of 24 (8 kv heads): 50 and 72; 64 of
  // 64 (4 kv heads), 6000 keys: 290 and 183; 112 of 24, 900 keys: 25.9 and 27.9, 6000 keys: 54
  // and 37.
  p->own_rows = each <= 48 || (length <= 1024 && heads * tiles16 <= room) ? 16 : 128;
  // And the prefix: narrow while that is half of a round of parts of 128 keys.  8 sequences of 32
  // heads (8 kv heads), 2000 keys: 15.1 us narrow, 20.5 wide; 16 of 32 (4 kv heads), 2000 keys,
  // twice that: 21.1 and 17.1.
  const int64_t most_prefix = (a.prefix_length + 127) / 128;
  p->prefix_rows =
      rows <= 16 || (p->own_rows == 16 && (rows + 15) / 16 * a.kv_heads * most_prefix <= room / 2)
          ? 16
          : 128;
  if (p->prefix_rows == 16) p->own_rows = 16;
  // workgroups, and keys that they read between them: about half of the bound
  int64_t own = 0, own_keys = 0;
  if (a.pages && a.n_indices && a.sequences) {
    int64_t tiles = (each + p->own_rows - 1) / p->own_rows;
    tiles = tiles < 4096 ? tiles : 4096;
    a.own_tiles = static_cast<int>(tiles);
    const int64_t units = tiles * heads;
    const int64_t most = (length + 127) / 128;
    // Lengths differ, so a round of parts of the bound is half empty: wide ones take a whole round
    // (24 sequences of 28 rows, 4000 keys: 110 us, 169 with half), narrow ones, whose loads
    // share the memory, half of one.  Where all run at once the longest would end alone, so long
    // ones are cut in any case, into three parts or more: 48 sequences, 8 kv heads, 4000 keys: 111
    // us, 161 without; 1800 keys: 60 and 80; but 1500 keys in two 62 to 85, 69 to 78 without.
    // More than run at once go in order of length instead, and cutting them costs: 128
    // sequences, 8 kv heads, 2048 keys: 138 us, 149 in three.  The order is for at most 256
    // sequences, one a thread (own_place): 128 of them 135 us, 152 as they come; 256 248 and 269;
    // 257, which go as they come, 274.
    int64_t splits = (p->own_rows == 16 ? room / 2 : room) / units;
    if (p->own_rows == 16 && units <= room && length > 1536 && splits < (length + 767) / 768)
      splits = (length + 767) / 768;
    splits = splits < 1 ? 1 : splits < most ? splits : most;
    const int64_t tile = p->own_rows == 16 ? 128 : 64;    // keys of a workgroup's turn
    a.own_chunk = static_cast<int>(up((length + splits - 1) / splits, tile));
    a.own_splits = static_cast<int>((length + a.own_chunk - 1) / a.own_chunk);
    a.sorted = units > room && a.sequences <= 256;
    own = units * a.own_splits;
    if (own > kMostWorkgroups) return refuse(-2, what, "2^24 workgroups or more", own);
    own_keys = units * length / 2;
  }
  a.prefix_tiles = static_cast<int>((rows + p->prefix_rows - 1) / p->prefix_rows);
  int64_t prefix = 0;
  if (a.prefix_length) {
    const int64_t units = static_cast<int64_t>(a.prefix_tiles) * a.kv_heads;
    // The prefix's parts are alike and start first, so they get the room that their share of the
    // keys to read asks for, and the own pages' take turns in the rest: their loads run beside the
    // prefix's products.  64 sequences of up to 4096 keys, 16384 shared: 184 us with a quarter of
    // the room, 227 with three; 128 of up to 2048, 32768 shared: 257 us with five eighths, 253
    // with six, 278 with all, 470 with two.  Own pages that are under an eighth of the work run
    // behind: 8 sequences on 131072 shared keys 112 us, 122 where they were given a quarter.
    const int64_t keys = units * a.prefix_length;
    const int64_t left =
        own_keys * 8 > own_keys + keys ? room - room * own_keys / (own_keys + keys) : room;
    int64_t splits = left == room ? room / units : (left + units / 2) / units;
    splits = splits < 1 ? 1 : splits < most_prefix ? splits : most_prefix;
    a.prefix_chunk = static_cast<int>(up((a.prefix_length + splits - 1) / splits, 128));
    // Parts of 128 keys, two tiles, while they are at most half a round, else at least four: 8
    // sequences of 32 heads (8 kv heads) on 8192 keys 19.0 us, 25.4 in a whole round of the
    // smallest parts; on 3000 keys 17.9 and 16.0.
    if (p->prefix_rows > 16 && a.prefix_chunk < 256 && units * most_prefix > room / 2)
      a.prefix_chunk = 256;
    a.prefix_splits = (a.prefix_length + a.prefix_chunk - 1) / a.prefix_chunk;
    prefix = units * a.prefix_splits;
  }
  a.slots = a.prefix_splits + a.own_splits;
  if ((prefix + 7) / 8 + (own + 7) / 8 > kMostWorkgroups / 8)
    return refuse(-2, what, "2^24 workgroups or more", prefix + own);
  a.prefix_eights = static_cast<int>((prefix + 7) / 8);
  a.own_eights = static_cast<int>((own + 7) / 8);
  p->bytes = static_cast<int64_t>(a.slots) * a.tokens * a.heads * (a.dim + 2) * 4;
  return 0;
}

template <typename T>
hipError_t launch_whole(const Plan& p, hipStream_t s) {
  if (p.a.dim <= 64) return launch_whole<T, 64>(p.a, s);
  if (p.a.dim <= 96) return launch_whole<T, 96>(p.a, s);
  if (p.a.dim <= 128) return launch_whole<T, 128>(p.a, s);
  return launch_whole<T, 256>(p.a, s);
}

template <typename T>
hipError_t launch_parts(const Plan& p, hipStream_t s) {
  if (p.a.dim <= 64) return launch_parts<T, 64>(p.a, p.prefix_rows, p.own_rows, s);
  if (p.a.dim <= 96) return launch_parts<T, 96>(p.a, p.prefix_rows, p.own_rows, s);
  if (p.a.dim <= 128) return launch_parts<T, 128>(p.a, p.prefix_rows, p.own_rows, s);
  return launch_parts<T, 256>(p.a, p.prefix_rows, p.own_rows, s);
}

template <typename T, int WAVES>
const void* join_of(int dim) {
  if (dim <= 64) return reinterpret_cast<const void*>(&join_parts<T, 16, WAVES>);
  if (dim <= 128) return reinterpret_cast<const void*>(&join_parts<T, 32, WAVES>);
  return reinterpret_cast<const void*>(&join_parts<T, 64, WAVES>);
}

template <typename T>
const void* join_of(int dim, bool shared) {
  return shared ? join_of<T, 4>(dim) : join_of<T, 1>(dim);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" __attribute__((visibility("default"))) int64_t prefix_attention_workspace(
    const tg_prefix_attention* r) {
  Plan p;
  if (const int rc = plan(r, &p)) return rc < 0 ? rc : -1;
  return p.bytes;
}

extern "C" __attribute__((visibility("default"))) int launch_prefix_attention(
    const tg_prefix_attention* r, void* stream) {
  const char* what = "launch_prefix_attention";
  Plan p;
  if (const int rc = plan(r, &p)) return rc;
  Attention& a = p.a;
  if (a.tokens == 0) return 0;
  if (!r->query || !r->out || !r->indptr || !r->lengths || (r->n_indices && !r->indices) ||
      (r->prefix_length && !r->prefix) || (r->pages && (!r->key_cache || !r->value_cache)))
    return refuse(-1, what, "null array", r->tokens);
  if (r->workspace_bytes < p.bytes || (p.bytes && !r->workspace))
    return refuse(-1, what, "the workspace is too small; bytes needed", p.bytes);
  if (reinterpret_cast<uintptr_t>(r->workspace) % 16)
    return refuse(-1, what, "the workspace is not 16-byte aligned", 0);
  const Operand query = {"query", r->query, 3, {r->tokens, r->heads, r->dim},
                         {r->query_token, r->query_head, 1}};
  const Operand out = {"out", r->out, 3, {r->tokens, r->heads, r->dim},
                       {r->out_token, r->out_head, 1}};
  const Operand kc = {"key_cache", r->key_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->kc_page, r->kc_slot, r->kc_head, 1}};
  const Operand vc = {"value_cache", r->value_cache, 4, {r->pages, r->page, r->kv_heads, r->dim},
                      {r->vc_page, r->vc_slot, r->vc_head, 1}};
  if (const int rc = once(what, out)) return rc;
  if (!same(out, query))
    if (const int rc = apart(what, out, query, 2)) return rc;
  for (const Operand* x : {&kc, &vc})
    if (const int rc = apart(what, out, *x, 2)) return rc;
  a.part = static_cast<float*>(r->workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part + static_cast<int64_t>(a.slots) * a.tokens *
                                                     a.heads * a.dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.whole) {
    const hipError_t e = r->dtype == TG_F16 ? launch_whole<_Float16>(p, s)
                                            : launch_whole<__bf16>(p, s);
    return e == hipSuccess ? 0 : hip_failed(e, what);
  }
  if (a.slots) {
    const hipError_t e = r->dtype == TG_F16 ? launch_parts<_Float16>(p, s)
                                            : launch_parts<__bf16>(p, s);
    if (e != hipSuccess) return hip_failed(e, what);
  }
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
  const bool shared = a.slots > 16 && rows <= kMostWorkgroups;
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(
      r->dtype == TG_F16 ? join_of<_Float16>(a.dim, shared) : join_of<__bf16>(a.dim, shared),
      dim3(static_cast<unsigned>(shared ? rows : (rows + 3) / 4)), dim3(256), args, 0, s);
  return e == hipSuccess ? 0 : hip_failed(e, what);
}
