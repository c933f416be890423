// Attention of new tokens over a paged cache, a block per query head: the form
// for every type, head size, page size and stride.
//
//   S_j = scale q . k_j for the keys j <= p, j > p - window, at p the token's
//   position;  O = sum_j exp(S_j - m) v_j / sum_j exp(S_j - m)
//
// in one pass over the keys with the running maximum m and sum.  Eight warps
// take every eighth group of four keys; a lane has every 32nd element of a
// head.  The warps' parts are joined through shared memory in warp order.  No
// key that the token does not see is read.  Bound by instructions, and by reading
// the cache once per query head: 64 tokens of 32 heads over contexts to 8192 took
// 3.1 ms, a prompt of 8192 216 ms, one token over 777 80 us (the tensor cores: 0.22,
// 0.63 and 0.017), all of 128 elements in bf16.  Elementary torch operations, which
// read a cache once per kv head, are slower for few tokens and faster for prompts:
// 16 tokens over contexts to 4096 f32 0.76 ms (1.1), bf16 heads of 256 1.4 (2.4);
// a prompt of 2048 f32 13 (3.1), bf16 heads of 256 28 (4.2).
#pragma once

#include <cmath>

#include "heads.cuh"

namespace ftb {

struct PagedAttentionParams {
  const void* q;  // [tokens, heads, dim]
  int64_t q_token, q_head;
  void* out;
  int64_t o_token, o_head;
  const void *keys, *values;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;
  PagedBatchParams batch;
  int tokens, heads, kv_heads, dim;
  int window;   // 0: none
  float scale;  // of the scores, times log2(e)
};

constexpr int kPagedRowsWarps = 8;

template <typename T, int NE>
__global__ void __launch_bounds__(32 * kPagedRowsWarps) paged_rows_kernel(const PagedAttentionParams p) {
  __shared__ float part[kPagedRowsWarps][32 * NE];
  __shared__ float stat[kPagedRowsWarps][2];
  grid_dep_wait();
  grid_dep_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (int)(blockIdx.x / p.heads), h = (int)(blockIdx.x % p.heads), kvh = h / (p.heads / p.kv_heads);
  int seq;
  int64_t position;
  if (!place_of(p.batch, t, lane, &seq, &position)) return;  // uniform over the block
  T* out = static_cast<T*>(p.out) + t * p.o_token + h * p.o_head;
  if (position >= (int64_t)p.batch.most_pages * p.batch.page_size) {  // beyond the table
    for (int e = threadIdx.x; e < p.dim; e += 32 * kPagedRowsWarps) out[e] = from_f32<T>(NAN);
    return;
  }
  const int* table = p.batch.page_table + seq * p.batch.table_ld;
  const int64_t first = p.window ? max((int64_t)0, position - p.window + 1) : 0;
  const T* q = static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head;
  float x[NE], o[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    x[i] = lane + 32 * i < p.dim ? to_f32(q[lane + 32 * i]) : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, sum = 0.0f;
  for (int64_t j0 = first + 4 * warp; j0 <= position; j0 += 4 * kPagedRowsWarps) {
    float s[4];
    const T* v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t j = j0 + c, n = j / p.batch.page_size;
      s[c] = 0.0f;
      v[c] = nullptr;
      if (j > position) continue;
      const int page = table[n];
      if (page < 0 || page >= p.batch.pages) continue;
      const int64_t in = j % p.batch.page_size;
      const T* k = static_cast<const T*>(p.keys) + page * p.k_page + in * p.k_token + kvh * p.k_head;
      v[c] = static_cast<const T*>(p.values) + page * p.v_page + in * p.v_token + kvh * p.v_head;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (lane + 32 * i < p.dim) s[c] = __fmaf_rn(x[i], to_f32(k[lane + 32 * i]), s[c]);
    }
    float top = m;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      for (int d = 16; d > 0; d >>= 1) s[c] += __shfl_xor_sync(0xffffffffu, s[c], d);
      s[c] *= p.scale;
      if (j0 + c > position) s[c] = -INFINITY;
      else if (!v[c]) s[c] = NAN;  // no such page
      top = fmaxf(top, s[c]);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    const float keep = exp2f(m - base);
    sum *= keep;
#pragma unroll
    for (int i = 0; i < NE; ++i) o[i] *= keep;
    m = top;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (j0 + c > position) continue;
      const float e = exp2f(s[c] - base);
      sum += e;
      if (!v[c]) continue;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (lane + 32 * i < p.dim) o[i] = __fmaf_rn(e, to_f32(v[c][lane + 32 * i]), o[i]);
    }
  }
  if (lane == 0) {
    stat[warp][0] = m;
    stat[warp][1] = sum;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) part[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, total = 0.0f;
  for (int w = 0; w < kPagedRowsWarps; ++w) top = fmaxf(top, stat[w][0]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int w = 0; w < kPagedRowsWarps; ++w) total += stat[w][1] * exp2f(stat[w][0] - base);
  for (int e = threadIdx.x; e < p.dim; e += 32 * kPagedRowsWarps) {
    float a = 0.0f;
    for (int w = 0; w < kPagedRowsWarps; ++w)
      if (stat[w][0] != -INFINITY || stat[w][1] != 0.0f) a += part[w][e] * exp2f(stat[w][0] - base);
    out[e] = from_f32<T>(position < 0 ? 0.0f : a / total);
  }
}

template <typename T>
cudaError_t launch_paged_rows_type(const PagedAttentionParams& p, cudaStream_t s) {
  const int64_t blocks = (int64_t)p.tokens * p.heads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return pdl_launch(p.dim <= 128 ? paged_rows_kernel<T, 4> : paged_rows_kernel<T, 16>, dim3((unsigned)blocks),
                    dim3(32 * kPagedRowsWarps), 0, s, p);
}

inline cudaError_t launch_paged_rows(const PagedAttentionParams& p, int type, cudaStream_t s) {
  if (type == FTB_F32) return launch_paged_rows_type<float>(p, s);
  if (type == FTB_F16) return launch_paged_rows_type<__half>(p, s);
  return launch_paged_rows_type<__nv_bfloat16>(p, s);
}

}  // namespace ftb
