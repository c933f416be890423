// C entry points of the operators around a decoder layer's attention and
// behind its logits (include/forgetune_b200.h): argument checks and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>

#include "forgetune_b200.h"
#include "heads.cuh"
#include "logprobs.cuh"
#include "op_common.hpp"
#include "paged_attention.cuh"
#include "paged_rows.cuh"

namespace ftb {

cudaError_t decoder_prepare() { return paged_attention_prepare(); }

constexpr int64_t kMaxTokens = int64_t(1) << 27, kMaxHeads = 4096, kMaxStride = int64_t(1) << 40;

static int64_t size_of(int64_t type) { return type == FTB_F32 ? 4 : 2; }
static bool vec4(const void* p, int64_t type) { return aligned(p, 4 * size_of(type)); }

// Memory of heads: the outer of tokens and heads as rows, the inner as their columns.
static Span span(const ftb_heads& x, int64_t tokens, int64_t heads, int64_t dim) {
  const int64_t e = size_of(x.type);
  const bool by_token = heads == 1 || tokens == 1 || x.token >= x.head;
  const int64_t rows = by_token ? tokens : heads, inner = by_token ? heads : tokens;
  return {static_cast<const char*>(x.data), rows, ((inner - 1) * (by_token ? x.head : x.token) + dim) * e,
          (by_token ? x.token : x.head) * e};
}
static Span flat(const void* p, int64_t bytes) { return {static_cast<const char*>(p), 1, bytes, 0}; }

static std::string check(const char* what, const ftb_heads& x, int64_t tokens, int64_t heads, int64_t dim) {
  if (!is_plain(x.type)) return std::string(what) + " must be float32, float16 or bfloat16";
  if (!aligned(x.data, size_of(x.type))) return std::string(what) + " is not aligned to its type";
  const bool by_token = heads == 1 || tokens == 1 || x.token >= x.head;
  const int64_t inner = by_token ? heads : tokens, in = by_token ? x.head : x.token;
  const int64_t outer = by_token ? tokens : heads, out = by_token ? x.token : x.head;
  if (x.token < 0 || x.head < 0 || x.token > kMaxStride || x.head > kMaxStride || (inner > 1 && in < dim) ||
      (outer > 1 && out < (inner - 1) * in + dim))
    return std::string(what) + " heads overlap, or a stride is out of range";
  return "";
}

static std::string check(const ftb_paged_cache& c) {
  if (!is_plain(c.type)) return "the cache must be float32, float16 or bfloat16";
  if (c.pages < 1 || c.pages > 0x7fffffff || c.page_size < 1 || c.page_size > kMaxTokens || c.kv_heads < 1 ||
      c.kv_heads > kMaxHeads || c.dim < 1 || c.dim > kHeadsMaxDim)
    return "the cache needs 1 <= pages, page_size, kv_heads (at most 4096) and dim (at most 512)";
  if (!aligned(c.keys, size_of(c.type)) || !aligned(c.values, size_of(c.type))) return "the cache is not aligned to its type";
  const int64_t st[6] = {c.k_page, c.k_token, c.k_head, c.v_page, c.v_token, c.v_head};
  for (int64_t x : st)
    if (x < 0 || x > kMaxStride) return "a stride of the cache is out of range";
  return "";
}
static int64_t cache_bytes(const ftb_paged_cache& c, int64_t page, int64_t token, int64_t head) {
  return ((c.pages - 1) * page + (c.page_size - 1) * token + (c.kv_heads - 1) * head + c.dim) * size_of(c.type);
}
// Whether places of the pool are apart: strides, from the smallest, each beyond what the ones before span.
static bool places_apart(const ftb_paged_cache& c, int64_t page, int64_t token, int64_t head) {
  std::pair<int64_t, int64_t> d[3] = {{page, c.pages}, {token, c.page_size}, {head, c.kv_heads}};
  std::sort(d, d + 3);
  int64_t extent = c.dim;
  for (const auto& x : d) {
    if (x.second == 1) continue;
    if (x.first < extent) return false;
    extent = (x.second - 1) * x.first + extent;
  }
  return true;
}

// Whether keys and values in one buffer never meet: alike in their strides, and side by side within one of them.
static bool pools_apart(const ftb_paged_cache& c) {
  if (c.k_page != c.v_page || c.k_token != c.v_token || c.k_head != c.v_head) return false;
  const int64_t st[3] = {c.k_page, c.k_token, c.k_head}, n[3] = {c.pages, c.page_size, c.kv_heads};
  const int64_t bytes = static_cast<const char*>(c.values) - static_cast<const char*>(c.keys);
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 1) continue;
    const int64_t ld = st[i] * size_of(c.type), d = (bytes % ld + ld) % ld;
    int64_t in = c.dim * size_of(c.type);
    bool rows = true;  // larger strides are whole numbers of these rows
    for (int k = 0; k < 3; ++k) {
      if (n[k] == 1 || k == i) continue;
      if (st[k] < st[i]) in += (n[k] - 1) * st[k] * size_of(c.type);
      else rows &= st[k] % st[i] == 0;
    }
    if (rows && d >= in && d + in <= ld) return true;
  }
  return false;
}

static std::string check(const ftb_paged_batch& b) {
  if (b.sequences < 1 || b.sequences > kMaxTokens || b.most_pages < 1 || b.most_pages > kMaxTokens ||
      (b.sequences > 1 && b.table_ld < b.most_pages) || b.table_ld < 0 || b.table_ld > kMaxStride)
    return "the page table needs at least one sequence and one page, and rows that do not overlap";
  if (!aligned(b.page_table, 4) || !aligned(b.starts, 4) || !aligned(b.lengths, 4))
    return "page_table, starts or lengths is not aligned to its type";
  return "";
}

static std::string check(const ftb_rotation& r, int64_t dim) {
  if (r.pairs < 0 || r.pairs > dim / 2) return "more frequencies than pairs in a head";
  if (r.pairs > 0 && !r.frequencies) return "frequencies is null";
  if (!aligned(r.frequencies, 8)) return "frequencies is not aligned to its type";
  if (!(r.eps >= 0.0)) return "eps must not be negative";
  return "";
}

static PagedBatchParams params(const ftb_paged_batch& b, const ftb_paged_cache& c) {
  PagedBatchParams p{};
  p.page_table = b.page_table;
  p.table_ld = b.table_ld;
  p.starts = b.starts;
  p.lengths = b.lengths;
  p.seqs = (int)b.sequences;
  p.most_pages = (int)b.most_pages;
  p.page_size = (int)c.page_size;
  p.pages = (int)c.pages;
  p.by_page = FastDiv((uint32_t)c.page_size);
  return p;
}

static void set_rotation(HeadsParams& p, const ftb_rotation& r) {
  p.frequencies = r.frequencies;
  p.pairs = (int)r.pairs;
  p.amplitude = r.amplitude;
  p.interleaved = r.interleaved != 0;
  p.norm = r.norm != 0;
  p.eps = (float)r.eps;
}

static void set_input(HeadsParams& p, int i, const ftb_heads& x, int64_t heads) {
  p.x[i] = x.data;
  p.x_token[i] = x.token;
  p.x_head[i] = x.head;
  p.heads[i] = (int)heads;
}

static bool in_fours(const ftb_heads& x) { return vec4(x.data, x.type) && x.token % 4 == 0 && x.head % 4 == 0; }

}  // namespace ftb

using namespace ftb;

FTB_API int ftb_rotate_heads(const ftb_rotate_args* args, void* stream) {
  static const char fn[] = "ftb_rotate_heads";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_rotate_args& a = *args;
    if (a.tokens == 0) return ST_OK;
    if (!a.x.data || !a.y.data || !a.positions) return refuse(fn, "null pointer", ST_NULL);
    if (a.tokens < 0 || a.tokens > kMaxTokens || a.heads < 1 || a.heads > kMaxHeads || a.dim < 1 ||
        a.dim > kHeadsMaxDim)
      return refuse(fn, "needs 0 <= tokens, 1 <= heads (at most 4096) and 1 <= dim (at most 512)");
    std::string why = check("x", a.x, a.tokens, a.heads, a.dim);
    if (why.empty()) why = check("y", a.y, a.tokens, a.heads, a.dim);
    if (why.empty() && a.x.type != a.y.type) why = "y must have x's type";
    if (why.empty()) why = check(a.rotation, a.dim);
    const int64_t pos = a.positions64 ? 8 : 4;
    if (why.empty() && (!aligned(a.positions, pos) || !aligned(a.weight, 4)))
      why = "positions or weight is not aligned to its type";
    if (why.empty()) {
      const Span x = span(a.x, a.tokens, a.heads, a.dim), y = span(a.y, a.tokens, a.heads, a.dim);
      const Span in[4] = {x, flat(a.positions, pos * a.tokens), flat(a.weight, 4 * a.dim),
                          flat(a.rotation.frequencies, 8 * a.rotation.pairs)};
      const bool in_place = a.x.data == a.y.data && (a.tokens == 1 || a.x.token == a.y.token) &&
                            (a.heads == 1 || a.x.head == a.y.head);
      why = clashes("y", y, in, in_place ? &x : nullptr);
    }
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    HeadsParams p{};
    set_input(p, 0, a.x, a.heads);
    p.y[0] = a.y.data;
    p.y_token[0] = a.y.token;
    p.y_head[0] = a.y.head;
    p.weight[0] = a.weight;
    set_rotation(p, a.rotation);
    p.tokens = (int)a.tokens;
    p.dim = (int)a.dim;
    p.positions = a.positions;
    p.positions64 = a.positions64 != 0;
    return launched(fn, launch_heads(p, (int)a.x.type, (int)a.x.type, in_fours(a.x) && in_fours(a.y), d->sm_count,
                                     static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_append_heads(const ftb_append_args* args, void* stream) {
  static const char fn[] = "ftb_append_heads";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_append_args& a = *args;
    const ftb_paged_cache& c = a.cache;
    if (a.tokens == 0) return ST_OK;
    if (!a.q.data || !a.k.data || !a.v.data || !a.q_out.data || !c.keys || !c.values || !a.batch.page_table ||
        !a.batch.starts || !a.batch.lengths)
      return refuse(fn, "null pointer", ST_NULL);
    if (a.tokens < 0 || a.tokens > kMaxTokens || a.heads < 1 || a.heads > kMaxHeads)
      return refuse(fn, "needs 0 <= tokens and 1 <= heads (at most 4096)");
    std::string why = check(c);
    if (why.empty()) why = check(a.batch);
    if (why.empty()) why = check("q", a.q, a.tokens, a.heads, c.dim);
    if (why.empty()) why = check("k", a.k, a.tokens, c.kv_heads, c.dim);
    if (why.empty()) why = check("v", a.v, a.tokens, c.kv_heads, c.dim);
    if (why.empty()) why = check("q_out", a.q_out, a.tokens, a.heads, c.dim);
    if (why.empty() && (a.q.type != a.k.type || a.q.type != a.v.type)) why = "q, k and v must have one type";
    if (why.empty() && a.q.type != c.type && a.q.type != FTB_F32) why = "q, k and v must have the cache's type or float32";
    if (why.empty() && a.q_out.type != c.type) why = "q_out must have the cache's type";
    if (why.empty()) why = check(a.rotation, c.dim);
    if (why.empty() && (!aligned(a.q_weight, 4) || !aligned(a.k_weight, 4))) why = "a weight is not aligned to its type";
    if (why.empty() && (!places_apart(c, c.k_page, c.k_token, c.k_head) || !places_apart(c, c.v_page, c.v_token, c.v_head)))
      why = "places of the cache overlap";
    if (why.empty()) {
      const Span q = span(a.q, a.tokens, a.heads, c.dim), out = span(a.q_out, a.tokens, a.heads, c.dim);
      const Span k = span(a.k, a.tokens, c.kv_heads, c.dim), v = span(a.v, a.tokens, c.kv_heads, c.dim);
      const Span keys = flat(c.keys, cache_bytes(c, c.k_page, c.k_token, c.k_head));
      const Span values = flat(c.values, cache_bytes(c, c.v_page, c.v_token, c.v_head));
      const Span in[9] = {q, k, v, flat(a.q_weight, 4 * c.dim), flat(a.k_weight, 4 * c.dim),
                          flat(a.rotation.frequencies, 8 * a.rotation.pairs),
                          span(a.batch.page_table, a.batch.sequences, 4 * a.batch.most_pages, 4 * a.batch.table_ld),
                          flat(a.batch.starts, 4 * (a.batch.sequences + 1)), flat(a.batch.lengths, 4 * a.batch.sequences)};
      const bool in_place = a.q.type == c.type && a.q.data == a.q_out.data &&
                            (a.tokens == 1 || a.q.token == a.q_out.token) && (a.heads == 1 || a.q.head == a.q_out.head);
      why = clashes("q_out", out, in, in_place ? &q : nullptr);
      if (why.empty()) why = clashes("keys", keys, in);
      if (why.empty()) why = clashes("values", values, in);
      if (why.empty() && (overlap(keys, out) || overlap(values, out))) why = "q_out overlaps the cache";
      if (why.empty() && overlap(keys, values) && !pools_apart(c)) why = "keys overlap values";
    }
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    HeadsParams p{};
    set_input(p, 0, a.q, a.heads);
    set_input(p, 1, a.k, c.kv_heads);
    set_input(p, 2, a.v, c.kv_heads);
    p.y[0] = a.q_out.data;
    p.y_token[0] = a.q_out.token;
    p.y_head[0] = a.q_out.head;
    p.y[1] = c.keys;
    p.y_page[1] = c.k_page;
    p.y_token[1] = c.k_token;
    p.y_head[1] = c.k_head;
    p.y[2] = c.values;
    p.y_page[2] = c.v_page;
    p.y_token[2] = c.v_token;
    p.y_head[2] = c.v_head;
    p.weight[0] = a.q_weight;
    p.weight[1] = a.k_weight;
    set_rotation(p, a.rotation);
    p.tokens = (int)a.tokens;
    p.dim = (int)c.dim;
    p.batch = params(a.batch, c);
    const bool vec = in_fours(a.q) && in_fours(a.k) && in_fours(a.v) && in_fours(a.q_out) && vec4(c.keys, c.type) &&
                     vec4(c.values, c.type) && c.k_page % 4 == 0 && c.k_token % 4 == 0 && c.k_head % 4 == 0 &&
                     c.v_page % 4 == 0 && c.v_token % 4 == 0 && c.v_head % 4 == 0;
    return launched(fn, launch_heads(p, (int)a.q.type, (int)c.type, vec, d->sm_count, static_cast<cudaStream_t>(stream)));
  });
}

namespace ftb {

static int check_attention(const char* fn, const ftb_attention_args& a) {
  const ftb_paged_cache& c = a.cache;
  if (!a.q.data || !a.out.data || !c.keys || !c.values || !a.batch.page_table || !a.batch.starts || !a.batch.lengths)
    return refuse(fn, "null pointer", ST_NULL);
  if (a.tokens < 0 || a.tokens > kMaxTokens || a.heads < 1 || a.heads > kMaxHeads)
    return refuse(fn, "needs 0 <= tokens and 1 <= heads (at most 4096)");
  std::string why = check(c);
  if (why.empty() && a.tokens * a.heads > 0x7fffffff) why = "tokens times heads must be below 2^31";
  if (why.empty() && a.heads % c.kv_heads) why = "heads must be a multiple of kv_heads";
  if (why.empty()) why = check(a.batch);
  if (why.empty()) why = check("q", a.q, a.tokens, a.heads, c.dim);
  if (why.empty()) why = check("out", a.out, a.tokens, a.heads, c.dim);
  if (why.empty() && (a.q.type != c.type || a.out.type != c.type)) why = "q, out and the cache must have one type";
  if (why.empty() && !(std::fabs(a.scale) * 1.4426950408889634 < 3.4e38)) why = "scale must be finite in float32, times log2(e) too";
  if (why.empty() && (a.window < 0 || a.window > 0x7fffffff)) why = "window must not be negative";
  if (why.empty()) {
    const Span in[6] = {span(a.q, a.tokens, a.heads, c.dim), flat(c.keys, cache_bytes(c, c.k_page, c.k_token, c.k_head)),
                        flat(c.values, cache_bytes(c, c.v_page, c.v_token, c.v_head)),
                        span(a.batch.page_table, a.batch.sequences, 4 * a.batch.most_pages, 4 * a.batch.table_ld),
                        flat(a.batch.starts, 4 * (a.batch.sequences + 1)), flat(a.batch.lengths, 4 * a.batch.sequences)};
    why = clashes("out", span(a.out, a.tokens, a.heads, c.dim), in);
  }
  return why.empty() ? (int)ST_OK : refuse(fn, why);
}

static PagedAttentionParams params(const ftb_attention_args& a) {
  const ftb_paged_cache& c = a.cache;
  PagedAttentionParams p{};
  p.q = a.q.data;
  p.q_token = a.q.token;
  p.q_head = a.q.head;
  p.out = a.out.data;
  p.o_token = a.out.token;
  p.o_head = a.out.head;
  p.keys = c.keys;
  p.values = c.values;
  p.k_page = c.k_page;
  p.k_token = c.k_token;
  p.k_head = c.k_head;
  p.v_page = c.v_page;
  p.v_token = c.v_token;
  p.v_head = c.v_head;
  p.batch = params(a.batch, c);
  p.tokens = (int)a.tokens;
  p.heads = (int)a.heads;
  p.kv_heads = (int)c.kv_heads;
  p.dim = (int)c.dim;
  p.window = (int)a.window;
  p.scale = (float)(a.scale * 1.4426950408889634);
  return p;
}

}  // namespace ftb

FTB_API int64_t ftb_paged_attention_workspace(const ftb_attention_args* args) {
  static const char fn[] = "ftb_paged_attention_workspace";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    if (args->tokens == 0) return 0;
    if (const int rc = check_attention(fn, *args)) return rc;
    const PagedAttentionParams p = params(*args);
    return paged_on_tensor_cores(p, (int)args->cache.type) ? (int)paged_workspace(p) : 0;
  });
}

FTB_API int ftb_paged_attention(const ftb_attention_args* args, void* stream) {
  static const char fn[] = "ftb_paged_attention";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_attention_args& a = *args;
    const ftb_paged_cache& c = a.cache;
    if (a.tokens == 0) return ST_OK;
    if (const int rc = check_attention(fn, a)) return rc;
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    const PagedAttentionParams p = params(a);
    const auto st = static_cast<cudaStream_t>(stream);
    if (!paged_on_tensor_cores(p, (int)c.type)) return launched(fn, launch_paged_rows(p, (int)c.type, st));
    if (a.workspace_bytes < paged_workspace(p) || !a.workspace || !aligned(a.workspace, 16))
      return refuse(fn, "needs the workspace that ftb_paged_attention_workspace tells, on 16-byte boundaries");
    return launched(fn, launch_paged_attention(p, (int)c.type, a.workspace, d->sm_count, d->fault_dev, op_stall(), st));
  });
}

FTB_API int ftb_token_logprobs(const ftb_logprobs_args* args, void* stream) {
  static const char fn[] = "ftb_token_logprobs";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_logprobs_args& a = *args;
    if (a.m == 0) return ST_OK;
    if (!a.logits.data || !a.tokens || !a.logprobs || !a.entropy || (a.top != 0 && (!a.top_logprobs || !a.top_tokens)))
      return refuse(fn, "null pointer", ST_NULL);
    if (a.m < 0 || a.m > kMaxTokens || a.n < 1 || a.n > kMaxTokens) return refuse(fn, "needs 0 <= m and 1 <= n, at most 2^27");
    if (a.top < 0 || a.top > kLogprobsMaxTop || a.top > a.n) return refuse(fn, "top must be 0 to 64 and at most n");
    std::string why = check("logits", a.logits, a.n);
    const int64_t size = a.tokens64 ? 8 : 4;
    if (why.empty() && (a.token_stride < 0 || a.token_stride > kMaxStride)) why = "token_stride is out of range";
    if (why.empty() && (!aligned(a.tokens, size) || !aligned(a.logprobs, 4) || !aligned(a.entropy, 4) ||
                        (a.top && (!aligned(a.top_logprobs, 4) || !aligned(a.top_tokens, 8)))))
      why = "tokens or an output is not aligned to its type";
    const Span in[2] = {span(a.logits, a.m, a.n), flat(a.tokens, ((a.m - 1) * a.token_stride + 1) * size)};
    const Span out[4] = {flat(a.logprobs, 4 * a.m), flat(a.entropy, 4 * a.m),
                         flat(a.top ? a.top_logprobs : nullptr, 4 * a.m * a.top),
                         flat(a.top ? a.top_tokens : nullptr, 8 * a.m * a.top)};
    for (int i = 0; i < 4 && why.empty(); ++i) {
      why = clashes("an output", out[i], in);
      for (int j = 0; j < i && why.empty(); ++j)
        if (overlap(out[i], out[j])) why = "outputs overlap";
    }
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    LogprobsParams p{};
    p.x = a.logits.data;
    p.ld = a.logits.ld;
    p.m = (int)a.m;
    p.n = (int)a.n;
    p.top = (int)a.top;
    p.tokens = a.tokens;
    p.tokens64 = a.tokens64 != 0;
    p.token_stride = a.token_stride;
    p.logprobs = a.logprobs;
    p.entropy = a.entropy;
    p.top_values = a.top_logprobs;
    p.top_tokens = a.top_tokens;
    return launched(fn, launch_logprobs(p, (int)a.logits.type, d->sm_count, static_cast<cudaStream_t>(stream)));
  });
}
