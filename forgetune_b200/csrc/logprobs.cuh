// Log probabilities of given tokens, the entropy of the distribution and its
// top alternatives, from rows of logits.
//
//   L = log sum_i exp(x_i),  logprob = x_token - L,  H = -sum_i p_i log p_i = L - sum_i p_i x_i
//
// in one pass over the row: with the running maximum m, s = sum exp(x - m) and
// t = sum exp(x - m) (x - m); when m grows by d, s and t become s e^-d and
// (t - s d) e^-d.  Then L = m + log s and H = log s - t / s.
//
// The alternatives come from the same pass.  The maxima of 64 disjoint parts
// of the row are values of it, so the k-th largest of them is at most the
// k-th largest value: only threads whose own maximum reaches it can hold one
// of the top k, and only their vectors are read again (from L2), by all
// threads at once.  What reaches the bound is ordered by value and, where equal, by
// index, as one 64-bit number, and ranked by counting.  Where too many values
// reach it (many equal ones), a bisection over the values finds the k-th.
//
// Bound by the logits' bytes, read once, and next to it by issue slots.  A block
// takes a row; of few rows a cluster of up to eight blocks takes one, and the
// first joins their sums and lists over distributed shared memory.
// In a graph of ten calls: 4096 x 131072 bf16 197 us (5.5 TB/s), 226 with 8
// alternatives (calls for longer, at the power limit, 250), 264 with 20; 333 x
// 50001 f16 12.1, and 17 with 20 (the ranking).  Rows of which four values are
// finite: 313 us without alternatives (0 times -inf sends every vector through the
// second sum), 307 with 3, 16 ms with 8 (the bisection).  Two vectors on their
// way and five blocks an SM took 268 us with 8 where four and three took 286 (two
// and four: 292); vectors inside of the row loaded without a check each, 226.
// 64 parts: with 256, 333 x 50001 with 20 took 34 us (17.8), by counting them.
#pragma once

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "fp8_format.cuh"
#include "tc_ptx.cuh"

namespace ftb {

constexpr int kLogprobsThreads = 256;
constexpr int kLogprobsParts = 64;  // at least the largest number of alternatives
constexpr int kLogprobsMaxTop = 64;
constexpr int kLogprobsCandidates = 1024;

struct LogprobsParams {
  const void* x;  // [m, n], rows ld apart
  int64_t ld;
  int m, n, top;
  const void* tokens;
  int tokens64;
  int64_t token_stride;
  float *logprobs, *entropy;
  float* top_values;     // [m, top]
  int64_t* top_tokens;
};

// Values in their order as whole numbers: zeros alike, NaN below all others.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Running sums of a part of a row; m stays finite from below.
struct RowSums {
  float m, s, t;
  __device__ __forceinline__ void raise(float top) {
    const float d = m - top;  // <= 0
    const float f = ex2(d * kLog2e);
    t = __fmaf_rn(s, fmaxf(d, -1e4f), t) * f;
    s *= f;
    m = top;
  }
  __device__ __forceinline__ void add(const RowSums& o) {
    RowSums b = o;
    const float top = fmaxf(m, b.m);
    raise(top);
    b.raise(top);
    s += b.s;
    t += b.t;
  }
};

// A plain load, after grid_dep_wait: the kernel before may have written the row after this one began, which the
// read-only loads do not allow.  (Written as a C++ load the compiler spilled 20 bytes a thread in place of 4:
// 4096 x 131072 with 8 alternatives 249 us in place of 240.)
__device__ __forceinline__ uint4 load_row(const uint4* p) {
  uint4 u;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}

template <typename T>
struct RowVectors {
  static constexpr int W = 16 / (int)sizeof(T);
  const T* row;
  int n, off, count;  // the row starts `off` elements into its first vector
  __device__ __forceinline__ RowVectors(const T* r, int size) : row(r), n(size) {
    off = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    count = (n + off + W - 1) / W;
  }
  __device__ __forceinline__ int first(int v) const { return v * W - off; }
  __device__ __forceinline__ bool whole(int v) const { return first(v) >= 0 && first(v) + W <= n; }
  // Vector v; what lies outside of the row reads as -inf.
  __device__ __forceinline__ uint4 load(int v) const {
    const int e = first(v);
    if (whole(v)) return load_row(reinterpret_cast<const uint4*>(row + e));
    T t[W];
#pragma unroll
    for (int i = 0; i < W; ++i) t[i] = e + i >= 0 && e + i < n ? row[e + i] : from_f32<T>(-INFINITY);
    uint4 u;
    memcpy(&u, t, 16);
    return u;
  }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float* f) {
  constexpr int W = 16 / (int)sizeof(T);
  T t[W];
  memcpy(t, &u, 16);
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = to_f32(t[i]);
}

struct LogprobsSmem {
  unsigned long long found[kLogprobsCandidates];
  unsigned long long best[kLogprobsMaxTop];  // in order
  alignas(16) uint32_t part[kLogprobsParts];
  RowSums sums[kLogprobsThreads / 32];
  RowSums total;
  int count, best_count, reach_count;
  uint16_t reach[kLogprobsThreads];  // threads whose maximum reaches the bound
  uint32_t bound;
};

// The k-th largest key of vectors [v0, v1) by bisection, then what is above it
// and, in order of index, of what equals it as much as is wanted.  All threads.
template <typename T>
__device__ __noinline__ void find_by_bisection(const RowVectors<T>& r, int v0, int v1, int k, LogprobsSmem& sm) {
  constexpr int W = RowVectors<T>::W;
  uint32_t lo = 0;  // at least k keys are >= lo
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t mid = lo | (1u << bit);
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    int c = 0;
    for (int v = v0 + threadIdx.x; v < v1; v += kLogprobsThreads) {
      float f[W];
      unpack<T>(r.load(v), f);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int e = r.first(v) + i;
        c += e >= 0 && e < r.n && order_key(f[i]) >= mid;
      }
    }
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) atomicAdd(&sm.count, c);
    __syncthreads();
    if (sm.count >= k) lo = mid;
  }
  __syncthreads();
  if (threadIdx.x == 0) sm.count = 0;
  __syncthreads();
  for (int v = v0 + threadIdx.x; v < v1; v += kLogprobsThreads) {
    float f[W];
    unpack<T>(r.load(v), f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int e = r.first(v) + i;
      const uint32_t key = order_key(f[i]);
      if (e >= 0 && e < r.n && key > lo)
        sm.found[atomicAdd(&sm.count, 1)] = (unsigned long long)key << 32 | (0xFFFFFFFFu - (uint32_t)e);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int have = sm.count;
    const int e0 = max(0, r.first(v0)), e1 = min(r.n, r.first(v1));
    for (int e = e0; e < e1 && have < k; e += 32) {
      const int i = e + (int)threadIdx.x;
      const bool hit = i < e1 && order_key(to_f32(r.row[i])) == lo;
      const uint32_t mask = __ballot_sync(0xffffffffu, hit);
      const int at = have + __popc(mask & ((1u << threadIdx.x) - 1u));
      if (hit && at < k) sm.found[at] = (unsigned long long)lo << 32 | (0xFFFFFFFFu - (uint32_t)i);
      have = min(k, have + __popc(mask));
    }
    __syncwarp();
    if (threadIdx.x == 0) sm.count = have;
  }
  __syncthreads();
}

// The k largest of found[0 .. count) into best, in order.  All threads.
__device__ __forceinline__ void rank_found(LogprobsSmem& sm, int k) {
  const int count = sm.count;
  for (int i = threadIdx.x; i < count; i += kLogprobsThreads) {
    const unsigned long long mine = sm.found[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += sm.found[j] > mine;
    if (rank < k) sm.best[rank] = mine;
  }
  if (threadIdx.x == 0) sm.best_count = min(k, count);
  __syncthreads();
}

// (s, t) += (a, b) (c, d)
__device__ __forceinline__ void row_fma2(float& s, float& t, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(s), "+f"(t)
      : "f"(a), "f"(b), "f"(c), "f"(d));
}
__device__ __forceinline__ float row_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kLogprobsThreads, 5) logprobs_kernel(const LogprobsParams p, const int split) {
  constexpr int W = RowVectors<T>::W, U = 2;
  __shared__ LogprobsSmem sm;
  grid_dep_wait();
  grid_dep_trigger();
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = (int)(blockIdx.x / split), rank = (int)(blockIdx.x % split);
  const RowVectors<T> r(static_cast<const T*>(p.x) + row * p.ld, p.n);
  const int v0 = (int)((int64_t)r.count * rank / split), v1 = (int)((int64_t)r.count * (rank + 1) / split);

  RowSums a{-FLT_MAX, 0.0f, 0.0f};
  float top = -INFINITY;
  uint4 u[U], next[U];
  const int whole0 = r.off ? 1 : 0, whole1 = min(v1, (r.n + r.off) / W);  // vectors inside of the row
  auto load = [&](uint4 (&to)[U], int v) {
    if (v >= whole0 && v + (U - 1) * kLogprobsThreads < whole1) {
      const uint4* from = reinterpret_cast<const uint4*>(r.row - r.off) + v;
#pragma unroll
      for (int i = 0; i < U; ++i) to[i] = load_row(from + i * kLogprobsThreads);
      return;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      T t[W];
#pragma unroll
      for (int k = 0; k < W; ++k) t[k] = from_f32<T>(-INFINITY);
      memcpy(&to[i], t, 16);
      if (v + i * kLogprobsThreads < v1) to[i] = r.load(v + i * kLogprobsThreads);
    }
  };
  load(next, v0 + tid);
  for (int v = v0 + tid; v < v1; v += U * kLogprobsThreads) {
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = next[i];
    load(next, v + U * kLogprobsThreads);  // on their way meanwhile
    float f[U][W], high[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < U; ++i) {
      unpack<T>(u[i], f[i]);
#pragma unroll
      for (int k = 0; k < W; k += 4) {
        high[0] = row_max3(high[0], f[i][k], f[i][k + 1]);
        high[1] = row_max3(high[1], f[i][k + 2], f[i][k + 3]);
      }
    }
    top = row_max3(top, high[0], high[1]);
    if (top > a.m) a.raise(top);
    float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < W; k += 2) {
        add2(f[i][k], f[i][k + 1], -a.m, -a.m);
        float x = f[i][k], y = f[i][k + 1];
        mul2(x, y, kLog2e, kLog2e);
        x = ex2(x);
        y = ex2(y);
        add2(s[0], s[1], x, y);
        row_fma2(t[0], t[1], x, y, f[i][k], f[i][k + 1]);
      }
    float more = t[0] + t[1];
    if (more != more) {  // 0 times -inf, unless something was NaN before
      more = 0.0f;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int k = 0; k < W; ++k) more = __fmaf_rn(ex2(f[i][k] * kLog2e), fmaxf(f[i][k], -1e4f), more);
    }
    a.s += s[0] + s[1];
    a.t += more;
  }
  const uint32_t mine = v0 + tid < v1 ? order_key(top) : 0u;

  for (int d = 16; d > 0; d >>= 1) {
    RowSums b{__shfl_xor_sync(0xffffffffu, a.m, d), __shfl_xor_sync(0xffffffffu, a.s, d),
              __shfl_xor_sync(0xffffffffu, a.t, d)};
    a.add(b);
  }
  if (lane == 0) sm.sums[warp] = a;
  constexpr int WIDTH = kLogprobsThreads / kLogprobsParts;
  uint32_t best = mine;
  for (int d = 1; d < WIDTH; d <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
  if (tid % WIDTH == 0) sm.part[tid / WIDTH] = best;
  if (tid == 0) sm.count = sm.reach_count = 0;
  __syncthreads();
  if (tid == 0) {
    RowSums all = sm.sums[0];
    for (int w = 1; w < kLogprobsThreads / 32; ++w) all.add(sm.sums[w]);
    sm.total = all;
  }
  const int e0 = max(0, r.first(v0)), e1 = min(p.n, r.first(v1)), k = min(p.top, e1 - e0);
  if (p.top > 0) {
    if (k > 0) {
      if (tid < kLogprobsParts) {
        const uint32_t key = sm.part[tid];
        const uint4* all = reinterpret_cast<const uint4*>(sm.part);
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < kLogprobsParts / 4; ++j) {
          const uint4 o = all[j];
          above += (o.x > key || (o.x == key && 4 * j < tid)) + (o.y > key || (o.y == key && 4 * j + 1 < tid)) +
                   (o.z > key || (o.z == key && 4 * j + 2 < tid)) + (o.w > key || (o.w == key && 4 * j + 3 < tid));
        }
        if (above == k - 1) sm.bound = key;
      }
      __syncthreads();
      const uint32_t bound = sm.bound;
      // the vectors of all threads that reach the bound, spread over the block
      if (v0 + tid < v1 && mine >= bound) sm.reach[atomicAdd(&sm.reach_count, 1)] = (uint16_t)tid;
      __syncthreads();
      const int each = (v1 - v0 + kLogprobsThreads - 1) / kLogprobsThreads, work = sm.reach_count * each;
#pragma unroll 2
      for (int w = tid; w < work; w += kLogprobsThreads) {
        const int q = w / each, v = v0 + sm.reach[q] + (w - q * each) * kLogprobsThreads;
        if (v >= v1) continue;
        float f[W];
        unpack<T>(r.load(v), f);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const int e = r.first(v) + i;
          const uint32_t key = order_key(f[i]);
          if (key >= bound && e >= 0 && e < p.n) {
            const int at = atomicAdd(&sm.count, 1);
            if (at < kLogprobsCandidates)
              sm.found[at] = (unsigned long long)key << 32 | (0xFFFFFFFFu - (uint32_t)e);
          }
        }
      }
      __syncthreads();
      if (sm.count > kLogprobsCandidates || sm.count < k) find_by_bisection<T>(r, v0, v1, k, sm);
      rank_found(sm, k);
    } else if (tid == 0) {
      sm.best_count = 0;
    }
  }
  if (split > 1) {
    cluster_sync_all();
    if (rank == 0) {
      if (tid == 0) {
        RowSums all = sm.total;
        for (int c = 1; c < split; ++c) {
          RowSums b;
          const uint32_t at = cluster_addr(&sm.total, c);
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.m) : "r"(at) : "memory");
          asm volatile("ld.shared::cluster.f32 %0, [%1 + 4];" : "=f"(b.s) : "r"(at) : "memory");
          asm volatile("ld.shared::cluster.f32 %0, [%1 + 8];" : "=f"(b.t) : "r"(at) : "memory");
          all.add(b);
        }
        sm.total = all;
        sm.count = 0;
      }
      __syncthreads();
      if (p.top > 0) {
        const int i = tid % kLogprobsMaxTop;  // eight lists of 64
        for (int c = tid / kLogprobsMaxTop; c < split; c += kLogprobsThreads / kLogprobsMaxTop) {
          int have;
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(have) : "r"(cluster_addr(&sm.best_count, c)) : "memory");
          if (i < have) {
            unsigned long long key;
            asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(cluster_addr(&sm.best[i], c)) : "memory");
            sm.found[atomicAdd(&sm.count, 1)] = key;
          }
        }
        __syncthreads();
        rank_found(sm, p.top);
      }
    }
    cluster_sync_all();  // no block leaves while its shared memory is read
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  const float m = sm.total.m, logs = logf(sm.total.s);
  auto logprob = [&](float x) { return (x - m) - logs; };
  if (tid == 0) {
    const int64_t at = row * p.token_stride;
    const int64_t token = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at];
    p.logprobs[row] = token >= 0 && token < p.n ? logprob(to_f32(r.row[token])) : __uint_as_float(0x7FC00000u);
    p.entropy[row] = logs - sm.total.t / sm.total.s;
  }
  for (int i = tid; i < p.top; i += kLogprobsThreads) {
    const unsigned long long key = sm.best[i];
    p.top_values[(int64_t)row * p.top + i] = logprob(key_value((uint32_t)(key >> 32)));
    p.top_tokens[(int64_t)row * p.top + i] = (int64_t)(0xFFFFFFFFu - (uint32_t)key);
  }
}

// Blocks per row: as many of up to eight as find an SM and 32 KB each.  us with 8 alternatives, one block in
// brackets: 1 x 32768 f32 6.9 (7.4), 16 x 131072 bf16 9.6 (16.4), 64 x 131072 12.3 (16.0).  With three blocks an SM and
// 8 KB: 100 x 131072 17.4 (16.2), 200 x 131072 25.2 (21.9), 1 x 8192 f32 with 5 6.2 (4.9).
inline int logprobs_split(int64_t m, int64_t bytes, int sm_count) {
  int split = 1;
  while (split < 8 && m * split * 2 <= sm_count && bytes / (2 * split) >= 32768) split *= 2;
  return split;
}

template <typename T>
cudaError_t launch_logprobs_type(const LogprobsParams& p, int sm_count, cudaStream_t s) {
  const int split = logprobs_split(p.m, (int64_t)p.n * (int64_t)sizeof(T), sm_count);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.m * (unsigned)split);
  cfg.blockDim = dim3(kLogprobsThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p, split);
}

inline cudaError_t launch_logprobs(const LogprobsParams& p, int type, int sm_count, cudaStream_t s) {
  if (type == FTB_F32) return launch_logprobs_type<float>(p, sm_count, s);
  if (type == FTB_F16) return launch_logprobs_type<__half>(p, sm_count, s);
  return launch_logprobs_type<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace ftb
