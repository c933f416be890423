// Heads of queries and keys turned by their tokens' positions, normalised
// first where asked, and keys and values stored into a paged cache.
//
//   n = x / sqrt(mean(x^2) + eps) w          over the head (or n = x)
//   a_i = position f_i,  c_i = A cos a_i,  s_i = A sin a_i
//   y_i = n_i c_i - n_j s_i,  y_j = n_j c_i + n_i s_i
//
// with pairs (i, j) = (i, i + r/2), or (2 i, 2 i + 1) where interleaved, over
// the first r elements of the head; the rest of it is n.  Angles are formed in
// 64 bits, reduced to a fraction of a turn there and passed on in 32: an angle
// of a million radians is then as exact as one of one radian.  The sum of
// squares, the norm and the rotation are fp32, and a value is rounded once.
//
// Bound by the bytes of x and y.  A lane holds V pairs of a head (two pieces
// of V elements: either side of the half, or side by side where interleaved),
// so no value crosses lanes but the sum of squares; up to 32 lanes share a head.
// A block takes a few tokens: it begins to load their heads, finds their
// sequences and pages and makes their cosines, once per token for all of its
// heads, then goes through the heads with the next ones on their way.
// In a graph of ten calls (calls in Python in brackets): 16384 x 16 x 128 f32 with
// the norm 55 us (59; 4.9 TB/s), 12725 tokens of 32 + 8 + 8 heads of 128 bf16
// appended with the norm 108 (108; 2.9 TB/s).  Both use two thirds of the issue
// slots, about 140 and 130 warp instructions for a head, which a head's 256 bytes
// in 16 bits need as 512 do in fp32.
#pragma once

#include <algorithm>
#include <cstring>

#include "fp8_format.cuh"
#include "tc_ptx.cuh"

namespace ftb {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsMaxDim = 512;

// n / d for 0 <= n < 2^31 by a product: with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1 it is
// (floor(m n / 2^32) + n) / 2^l (Granlund and Montgomery's division by invariant integers).
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t by) : d(by), mul(0), shift(0) {
    while (((uint64_t)1 << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int of(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

// New tokens of several sequences and the pages that hold them.
struct PagedBatchParams {
  const int* page_table;  // [seqs, most_pages], rows table_ld apart
  int64_t table_ld;
  const int* starts;      // [seqs + 1] first row of each sequence
  const int* lengths;     // [seqs] tokens with the new ones
  int seqs, most_pages, page_size, pages;
  FastDiv by_page;
};

// Number of entries <= t among starts[0 .. n), by a whole warp (32 blocks a step).
__device__ __forceinline__ int count_not_above(const int* starts, int n, int t, int lane) {
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) >> 5, i = lo + (lane + 1) * step - 1;
    const int c = __popc(__ballot_sync(0xffffffffu, (lane + 1) * (int64_t)step <= n && starts[i] <= t));
    lo += c * step;
    n = min(step, n - c * step);
    if (step == 1) break;
  }
  return lo;
}

// Sequence and position of row t; false where it belongs to none.
__device__ __forceinline__ bool place_of(const PagedBatchParams& b, int t, int lane, int* seq, int64_t* position) {
  const int s = count_not_above(b.starts, b.seqs + 1, t, lane) - 1;
  *seq = s;
  if (s < 0 || s >= b.seqs) return false;
  *position = (int64_t)b.lengths[s] - b.starts[s + 1] + t;
  return true;
}

struct HeadsParams {
  const void* x[3];  // q, k, v [tokens, heads, dim]
  int64_t x_token[3], x_head[3];
  int heads[3];
  void* y[3];        // q's output; the pool of keys, of values
  int64_t y_token[3], y_head[3], y_page[3];
  const float* weight[2];
  float eps;
  int norm;
  const double* frequencies;
  int pairs;         // r / 2
  double amplitude;
  int interleaved;
  int tokens, dim;
  const void* positions;  // of each token, or null: from the batch
  int positions64;
  PagedBatchParams batch;
  int units, lanes;       // units of V pairs in a head, lanes that share them
  int per_block;          // heads of a token that a block takes
  int tokens_per_block, blocks_per_token;
  FastDiv by_pairs;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};

// One of the two pieces of unit u: its first element.
template <int V>
__device__ __forceinline__ void unit_at(const HeadsParams& p, int u, int* a, int* b) {
  const int turned = p.pairs / V;
  if (u >= turned) {
    *a = 2 * p.pairs + (u - turned) * 2 * V;
    *b = *a + V;
  } else if (p.interleaved) {
    *a = 2 * u * V;
    *b = *a + V;
  } else {
    *a = u * V;
    *b = *a + p.pairs;
  }
}

// V cosines and sines, which for V = 4 lie on a 16-byte boundary (pairs are a multiple of four).
template <int V>
__device__ __forceinline__ void load_turns(const float2* from, float2 (&to)[V]) {
  if constexpr (V == 4) {
    const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
    to[0] = make_float2(a.x, a.y), to[1] = make_float2(a.z, a.w), to[2] = make_float2(b.x, b.y), to[3] = make_float2(b.z, b.w);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = from[e];
  }
}

// AHEAD heads are on their way (and 28 bytes of a lane in fp32, 4 in bf16 are
// spilled for it).  Two, four blocks an SM: 55 us for the rotation above, 108 for the append; three: 58 and
// 106; two with five blocks 65 and 140; three with three 57 and 128; four with three 57 and 127.
template <typename T, typename O, int V, int UPL, int AHEAD>
__global__ void __launch_bounds__(kHeadsThreads, UPL == 1 ? 4 : 1) heads_kernel(const HeadsParams p) {
  extern __shared__ float4 turn4[];  // [tokens of the block][pairs] cosine and sine
  float2* turn = reinterpret_cast<float2*>(turn4);
  __shared__ int64_t where[64];      // position of a token
  __shared__ int64_t slot[2][64];    // where its key and value go
  __shared__ int page_of[64];        // its page; -1: no place in the pool, -2: no sequence
  grid_dep_wait();
  grid_dep_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = (int)(blockIdx.x / p.blocks_per_token) * p.tokens_per_block;
  const int h0 = (int)(blockIdx.x % p.blocks_per_token) * p.per_block;
  const int all = p.heads[0] + p.heads[1] + p.heads[2];
  const int group = threadIdx.x / p.lanes, groups = kHeadsThreads / p.lanes, l = threadIdx.x % p.lanes;
  const int tokens = min(p.tokens_per_block, p.tokens - t0);
  // A group of lanes takes one head of every token, or of every side-th, and then its next head.
  const int wide = min(p.per_block, groups), side = groups / wide, first = group / wide;
  const int turns = (p.per_block + wide - 1) / wide, steps = (tokens + side - 1) / side;

  // this lane's two pieces of each unit, in elements of the head; -1: none
  int at[UPL][2];
#pragma unroll
  for (int j = 0; j < UPL; ++j) {
    unit_at<V>(p, l + j * p.lanes, &at[j][0], &at[j][1]);
    if (l + j * p.lanes >= p.units) at[j][0] = at[j][1] = -1;
    else if (at[j][1] >= p.dim) at[j][1] = -1;
  }
  int kind = -1, head = 0, coming = 0;  // q, k, v or -1; the token of the next load
  const T* src = nullptr;
  int64_t stride = 0;
  auto begin = [&](int n) {  // its n-th head
    head = n * wide + group % wide;
    kind = first < side && head < p.per_block && h0 + head < all ? 0 : -1;
    head += h0;
    if (kind == 0 && head >= p.heads[0]) {
      head -= p.heads[0];
      kind = 1;
      if (head >= p.heads[1]) {
        head -= p.heads[1];
        kind = 2;
      }
    }
    const int k = max(kind, 0);
    src = static_cast<const T*>(p.x[k]) + (int64_t)(t0 + first) * p.x_token[k] + head * p.x_head[k];
    stride = side * p.x_token[k];
    coming = kind < 0 ? tokens : first;
  };
  auto load = [&](Piece<T, V> (&to)[UPL][2]) {  // of its next token; pieces that are not there stay zero
    if (coming < tokens) {
#pragma unroll
      for (int j = 0; j < UPL; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (at[j][s] >= 0) to[j][s] = *reinterpret_cast<const Piece<T, V>*>(src + at[j][s]);
    }
    src += stride;
    coming += side;
  };
  Piece<T, V> in[AHEAD][UPL][2];
  memset(in, 0, sizeof(in));
  begin(0);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(in[i]);

  for (int i = warp; i < tokens; i += kHeadsThreads / 32) {
    const int t = t0 + i;
    int64_t position = 0, to = 0;
    int page = -2;
    if (p.positions) {
      position = p.positions64 ? static_cast<const int64_t*>(p.positions)[t] : static_cast<const int*>(p.positions)[t];
      page = -1;
    } else {
      int seq;
      if (place_of(p.batch, t, lane, &seq, &position)) {
        const int n = position >= 0 ? p.batch.by_page.of((int)position) : p.batch.most_pages;
        page = n < p.batch.most_pages ? p.batch.page_table[seq * p.batch.table_ld + n] : -1;
        if (page < 0 || page >= p.batch.pages) page = -1;
        to = position - (int64_t)n * p.batch.page_size;
      }
    }
    if (lane == 0) {
      where[i] = position;
      page_of[i] = page;
      slot[0][i] = page * p.y_page[1] + to * p.y_token[1];
      slot[1][i] = page * p.y_page[2] + to * p.y_token[2];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * p.pairs; i += kHeadsThreads) {
    const int tok = p.by_pairs.of(i);
    // a / 2 pi in turns; what is left of whole turns is at most half a turn
    double a = (double)where[tok] * p.frequencies[i - tok * p.pairs] * 0.15915494309189535;
    a -= rint(a);
    float s, c;
    sincospif((float)(2.0 * a), &s, &c);
    turn[i] = make_float2((float)(p.amplitude * c), (float)(p.amplitude * s));
  }
  __syncthreads();

#pragma unroll 1
  for (int n = 0; n < turns; ++n) {
    const bool turned = kind == 0 || kind == 1;
    float w[UPL][2][V];  // the head's weights
#pragma unroll
    for (int j = 0; j < UPL; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < V; ++e) w[j][s][e] = turned && p.weight[kind] && at[j][s] >= 0 ? p.weight[kind][at[j][s] + e] : 1.0f;
    const int k = max(kind, 0);
    O* y = static_cast<O*>(p.y[k]) + head * p.y_head[k];
    if (kind == 0) y += (int64_t)(t0 + first) * p.y_token[0];
    int tok = first;
#pragma unroll 1
    for (int step = 0; step < steps; ++step, tok += side) {
      float v[UPL][2][V];
#pragma unroll
      for (int j = 0; j < UPL; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int e = 0; e < V; ++e) v[j][s][e] = to_f32(in[0][j][s].v[e]);
#pragma unroll
      for (int i = 0; i + 1 < AHEAD; ++i) memcpy(&in[i], &in[i + 1], sizeof(in[0]));
      load(in[AHEAD - 1]);
      if (p.norm) {  // whole warps: lanes of other kinds take part
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < UPL; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < V; ++e) sum = __fmaf_rn(v[j][s][e], v[j][s][e], sum);
        for (int d = p.lanes >> 1; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float r = turned ? rsqrtf(__fmaf_rn(sum, 1.0f / (float)p.dim, p.eps)) : 1.0f;
#pragma unroll
        for (int j = 0; j < UPL; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][s][e] = v[j][s][e] * r * w[j][s][e];
      }
      if (kind < 0 || tok >= tokens) continue;
      const int page = page_of[tok];
      if (page == -2 || (kind > 0 && page < 0)) continue;
      O* to = kind == 0 ? y + (int64_t)(step * side) * p.y_token[0] : y + slot[kind - 1][tok];
#pragma unroll
      for (int j = 0; j < UPL; ++j) {
        const int u = l + j * p.lanes;
        if (turned && u < p.pairs / V) {
          float2 q[V];
          load_turns<V>(turn + tok * p.pairs + u * V, q);
          if (p.interleaved && V > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) {  // pair e of the unit: elements 2 e and 2 e + 1 of the two pieces
              float& m = v[j][2 * e / V][2 * e % V];
              float& z = v[j][2 * e / V][2 * e % V + 1 < V ? 2 * e % V + 1 : 0];
              const float x = __fmaf_rn(m, q[e].x, -__fmul_rn(z, q[e].y));
              z = __fmaf_rn(z, q[e].x, __fmul_rn(m, q[e].y));
              m = x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float m = v[j][0][e], z = v[j][1][e];
              v[j][0][e] = __fmaf_rn(m, q[e].x, -__fmul_rn(z, q[e].y));
              v[j][1][e] = __fmaf_rn(z, q[e].x, __fmul_rn(m, q[e].y));
            }
          }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          Piece<O, V> out;
#pragma unroll
          for (int e = 0; e < V; ++e) out.v[e] = from_f32<O>(v[j][s][e]);
          if (at[j][s] >= 0) *reinterpret_cast<Piece<O, V>*>(to + at[j][s]) = out;
        }
      }
    }
    if (n + 1 < turns) {
      begin(n + 1);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) load(in[i]);
    }
  }
}

template <typename T, typename O, int V, int UPL, int AHEAD>
cudaError_t launch_heads_as(HeadsParams p, int sm_count, cudaStream_t s) {
  p.units = p.pairs / V + (p.dim - 2 * p.pairs + 2 * V - 1) / (2 * V);
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < p.units) p.lanes *= 2;
  const int groups = kHeadsThreads / p.lanes, all = p.heads[0] + p.heads[1] + p.heads[2];
  // few heads: a turn of the groups each; else whole tokens, as many as leave eight blocks for each SM, with cosines
  // in at most 16 KB.  us where few (and as many): 1 x 32 heads 3.2 (4.4), 16 tokens appended 3.9 (6.3); where many (and
  // as few): 16384 x 16 x 128 f32 55 (102), 12725 tokens appended 108 (242)
  const bool few = (int64_t)p.tokens * ((all + groups - 1) / groups) <= 4 * sm_count;
  p.per_block = few ? std::min(all, groups) : all;
  p.blocks_per_token = (all + p.per_block - 1) / p.per_block;
  const int fill = std::max(1, groups / p.per_block);  // tokens that a turn of the groups takes
  const int most = std::min(64, p.pairs ? std::max(1, 2048 / p.pairs) : 64);
  p.tokens_per_block = std::min(most, few ? fill : std::max(fill, std::min(p.tokens / (8 * sm_count), 8 * fill)));
  p.by_pairs = FastDiv((uint32_t)std::max(1, p.pairs));
  const int64_t blocks = ((int64_t)p.tokens + p.tokens_per_block - 1) / p.tokens_per_block * p.blocks_per_token;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return pdl_launch(heads_kernel<T, O, V, UPL, AHEAD>, dim3((unsigned)blocks), dim3(kHeadsThreads),
                    ((size_t)p.tokens_per_block * p.pairs * sizeof(float2) + 15) / 16 * 16, s, p);
}

// `vec`: every base and stride is a multiple of four elements.  Vectors also
// need dim and r in multiples of eight.  The form without them has the room for
// any head: 16384 x 16 x 128 bf16 off by one element takes 250 us, on a boundary
// 52; heads of 72 with 36 turned 236.
template <typename T, typename O>
cudaError_t launch_heads_types(const HeadsParams& p, bool vec, int sm_count, cudaStream_t s) {
  if (!vec || p.dim % 8 || p.pairs % 4) return launch_heads_as<T, O, 1, 8, 1>(p, sm_count, s);
  if (p.dim > 256) return launch_heads_as<T, O, 4, 2, 1>(p, sm_count, s);
  return launch_heads_as<T, O, 4, 1, 2>(p, sm_count, s);
}

inline cudaError_t launch_heads(const HeadsParams& p, int in, int out, bool vec, int sm_count, cudaStream_t s) {
  if (in == FTB_F32) {
    if (out == FTB_F32) return launch_heads_types<float, float>(p, vec, sm_count, s);
    if (out == FTB_F16) return launch_heads_types<float, __half>(p, vec, sm_count, s);
    return launch_heads_types<float, __nv_bfloat16>(p, vec, sm_count, s);
  }
  if (in == FTB_F16) return launch_heads_types<__half, __half>(p, vec, sm_count, s);
  return launch_heads_types<__nv_bfloat16, __nv_bfloat16>(p, vec, sm_count, s);
}

}  // namespace ftb
