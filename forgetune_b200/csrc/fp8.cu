// C entry points of the block-scaled 8-bit operators
// (include/forgetune_b200.h): argument checks, the per-device set-up and the
// launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

#include "forgetune_b200.h"
#include "fp8_gemm.cuh"
#include "fp8_pair.cuh"
#include "fp8_rows.cuh"
#include "op_common.hpp"
#include "rms_norm.hpp"

namespace ftb {

constexpr int kFp8MaxDevices = 64;
constexpr int64_t kFp8MaxDim = int64_t(1) << 27;

static OpDevice g_fp8_devices[kFp8MaxDevices];
static std::atomic<int> g_fp8_stall{0};  // failure-detection hook
static std::atomic<int> g_fp8_kernel{-1};  // kernel hook: 16 nt + split, or -1 for the estimate's choice

// Once per device; "" when done.  Allocates a word and sets kernel attributes,
// in relaxed capture mode, so that a stream under capture does not matter.
static std::string fp8_setup(int dev, OpDevice* d) {
  int major = 0;
  cudaError_t e = cudaDeviceGetAttribute(&d->sm_count, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess && major != 10) return "needs a GPU of compute capability 10.0 (sm_100a)";
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (e == cudaSuccess) e = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e == cudaSuccess) {
    if (!d->fault) {
      void *h = nullptr, *hd = nullptr;
      e = cudaHostAlloc(&h, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
      if (e == cudaSuccess) {
        *static_cast<int*>(h) = 0;
        e = cudaHostGetDevicePointer(&hd, h, 0);
        if (e == cudaSuccess) {
          d->fault = static_cast<volatile int*>(h);
          d->fault_dev = static_cast<int*>(hd);
        } else {
          cudaFreeHost(h);
        }
      }
    }
    if (e == cudaSuccess) e = fp8_tile_attributes<16>();
    if (e == cudaSuccess) e = fp8_tile_attributes<32>();
    if (e == cudaSuccess) e = fp8_tile_attributes<64>();
    if (e == cudaSuccess) e = fp8_tile_attributes<128>();
    if (e == cudaSuccess) e = fp8_pair_prepare(&d->pairs);
    if (e == cudaSuccess) e = decoder_prepare();
    const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaSuccess) e = back;
  }
  if (e == cudaSuccess) return "";
  cudaGetLastError();
  return std::string("set-up failed: ") + cudaGetErrorString(e);
}

int op_stall() { return g_fp8_stall.load(); }

int op_device(const char* fn, OpDevice** out) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return refuse(fn, cudaGetErrorString(e), ST_DEVICE);
  }
  if (dev < 0 || dev >= kFp8MaxDevices) return refuse(fn, "device ordinal beyond the supported range", ST_CONFIG);
  OpDevice& d = g_fp8_devices[dev];
  if (!d.ready.load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(d.mu);
    if (!d.ready.load(std::memory_order_relaxed)) {
      const std::string why = fp8_setup(dev, &d);
      if (!why.empty()) return refuse(fn, why, ST_DEVICE);
      d.ready.store(true, std::memory_order_release);
    }
  }
  // taken by one caller: of threads that find it at once, the others go on
  const int code = *d.fault != 0 ? __atomic_exchange_n(const_cast<int*>(d.fault), 0, __ATOMIC_RELAXED) : 0;
  if (code != 0)
    return refuse(fn, "an earlier call's kernel on this device gave up: a wait exceeded its limit (code " +
                          std::to_string(code) + "); that call's output is not valid", ST_DEVICE);
  *out = &d;
  return ST_OK;
}

static std::string check(const char* what, const ftb_fp8_matrix& q, int64_t cols) {
  if (!aligned(q.data, 16) || q.ld % 16 || q.ld < cols)
    return std::string(what) + " values need 16-byte aligned rows (base and stride) of at least their length";
  if (!aligned(q.scales, 4) || q.scales_ld % 4 || q.scales_ld < fp8_blocks(cols))
    return std::string(what) + " scales need 4-byte aligned rows (base and stride) of at least their length";
  return "";
}

// A quantised output of m rows and `scale_rows` rows of scales: over an operand,
// or the one over the other.
template <size_t N>
static std::string clashes(const char* what, const ftb_fp8_matrix& q, int64_t m, int64_t scale_rows, int64_t k,
                           const Span (&in)[N]) {
  const Span values = span(q.data, m, k, q.ld), scales = span(q.scales, scale_rows, fp8_blocks(k), q.scales_ld);
  std::string why = clashes(what, values, in);
  if (why.empty()) why = clashes(what, scales, in);
  if (why.empty() && overlap(values, scales)) why = std::string(what) + " scales overlap its values";
  return why;
}

static bool sizes_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && m <= kFp8MaxDim && n >= 1 && n <= kFp8MaxDim && k >= 1 && k <= kFp8MaxDim;
}

// The kernel for a product: the tile kernel with NT tokens per tile and a
// cluster of `split` CTAs per tile, or the pair kernel (nt = 0).
struct Fp8Choice {
  int nt, split;
};

// Picks by an estimate of the time in microseconds.  A round of the tile
// kernel's CTAs takes 0.31 per k-block (paid in series: the same with one CTA on
// the GPU as with many, and with rings of three, four and five stages), at least
// 0.0097 per KB that an SM's CTAs load, and 0.017 per token of a tile plus
// 0.013 per token of the SM for its epilogue; each CTA of an SM costs 0.23, a
// later round 1.3, a cluster 0.4.  A round is counted as two CTAs per SM, fewer
// in clusters of 4 and 8, which do not fill the SMs' groups: what registers and
// shared memory leave room for, but for 16 and 32 tokens unsplit, of which three
// fit.  There it counts rounds that do not happen: most of the worst picks below
// take 64 or 128 tokens where 32 unsplit is best.  A round of pairs takes 0.29
// per k-block and 0.8, and a launch 3.5 more than the tile kernel's.  The
// constants are a fit to 525 shapes (m 1..4096, n and k 64..8192) that were
// timed with every choice on a B200; over 696 others the pick is 1.1 % slower
// than the best choice in the mean, 28 % at most.  For example (m x k x n): 1 x
// 4096 x 4096 takes 5.0 us with 16 tokens per tile and split 4, 11.8 unsplit;
// 512 x 512 x 512 takes 3.3 with 16 tokens, 6.9 with 128; 256 x 4096 x 4096
// 11.9 with 128 tokens and split 2, 15.2 on pairs; 1024 x 4096 x 4096 16.6 on
// pairs, 22.3 with 128 tokens.
static Fp8Choice choose_fp8(int64_t m, int64_t n, int64_t k, const OpDevice& d) {
  static const double kResident[4] = {2.0, 2.0, 1.78, 1.73};  // CTAs per SM in clusters of 1, 2, 4 and 8
  const int64_t nk = fp8_blocks(k), tiles_n = fp8_blocks(n);
  const double pair_tiles = (double)((m + 255) / 256) * (double)((n + 255) / 256);
  Fp8Choice best{0, 1};
  double best_us = 5.19 + std::ceil(pair_tiles / d.pairs) * ((double)nk * 0.293 + 0.77);
  for (int nt = 16; nt <= 128; nt *= 2) {
    const double tiles = (double)tiles_n * (double)((m + nt - 1) / nt);
    for (int i = 0, split = 1; i < 4; ++i, split *= 2) {
      if (split > 1 && nk < split * 2) break;  // CTAs without a k-block
      const double ctas = tiles * split;
      const double kb = (double)std::min<int64_t>(nk, ((nk + 3) / 4 + split - 1) / split * 4);
      const double rounds = std::ceil(ctas / (kResident[i] * d.sm_count)), per_sm = std::ceil(ctas / d.sm_count);
      const double load = std::max(rounds * kb * 0.308, per_sm * kb * (16 + nt / 8) * 0.0097);
      const double us = 1.71 + load + nt * (rounds * 0.0168 + per_sm * 0.0126) + per_sm * 0.23 +
                        (rounds - 1) * 1.26 + (split > 1 ? 0.39 : 0.0);
      if (us < best_us) {
        best_us = us;
        best = Fp8Choice{nt, split};
      }
    }
    if (nt >= m) break;  // wider tiles would have empty columns only
  }
  return best;
}

static cudaError_t launch_fp8_linear(const Fp8Operands& o, const Fp8Params& p, const OpDevice& d, cudaStream_t s) {
  const int set = g_fp8_kernel.load(std::memory_order_relaxed);
  const Fp8Choice c = set < 0 ? choose_fp8(p.M, p.N, p.K, d) : Fp8Choice{set / 16, set % 16};
  switch (c.nt) {
    case 16: return launch_fp8_tile<16>(o, p, c.split, s);
    case 32: return launch_fp8_tile<32>(o, p, c.split, s);
    case 64: return launch_fp8_tile<64>(o, p, c.split, s);
    case 128: return launch_fp8_tile<128>(o, p, c.split, s);
    default: return launch_fp8_pair(o, p, d.pairs, s);
  }
}

cudaError_t rms_norm_f32(const float* x, const float* weight, float eps, float* y, int64_t m, int64_t k, int sm_count,
                         cudaStream_t s) {
  RowsParams p{};
  p.x = x;
  p.x_ld = k;
  p.weight = weight;
  p.eps = eps;
  p.y = y;
  p.y_ld = k;
  p.m = m;
  p.k = k;
  return launch_rms_norm(p, FTB_F32, sm_count, s);
}

}  // namespace ftb

using namespace ftb;

FTB_API int ftb_quantize_rows(const ftb_quantize_args* args, void* stream) {
  static const char fn[] = "ftb_quantize_rows";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_quantize_args& a = *args;
    if (a.m == 0) return ST_OK;
    if (!a.x.data || !a.q.data || !a.q.scales) return refuse(fn, "null pointer", ST_NULL);
    if (!sizes_ok(a.m, 1, a.k)) return refuse(fn, "needs 0 <= m and 1 <= k, at most 2^27");
    std::string why = check("x", a.x, a.k);
    if (why.empty()) why = check("q", a.q, a.k);
    const Span in[1] = {span(a.x, a.m, a.k)};
    if (why.empty()) why = clashes("q", a.q, a.m, a.m, a.k, in);
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = a.x.data;
    p.x_ld = a.x.ld;
    p.q = a.q.data;
    p.q_ld = a.q.ld;
    p.s = a.q.scales;
    p.s_ld = a.q.scales_ld;
    p.m = a.m;
    p.k = a.k;
    return launched(fn, launch_quantize_rows(p, (int)a.x.type, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_quantize_weight(const ftb_quantize_args* args, void* stream) {
  static const char fn[] = "ftb_quantize_weight";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_quantize_args& a = *args;
    if (a.m == 0) return ST_OK;
    if (!a.x.data || !a.q.data || !a.q.scales) return refuse(fn, "null pointer", ST_NULL);
    if (!sizes_ok(a.m, 1, a.k) || fp8_blocks(a.m) > 65535)
      return refuse(fn, "needs 0 <= m <= 128 * 65535 and 1 <= k <= 2^27");
    std::string why = check("x", a.x, a.k);
    if (why.empty()) why = check("q", a.q, a.k);
    const Span in[1] = {span(a.x, a.m, a.k)};
    if (why.empty()) why = clashes("q", a.q, a.m, fp8_blocks(a.m), a.k, in);
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = a.x.data;
    p.x_ld = a.x.ld;
    p.q = a.q.data;
    p.q_ld = a.q.ld;
    p.s = a.q.scales;
    p.s_ld = a.q.scales_ld;
    p.m = a.m;
    p.k = a.k;
    return launched(fn, launch_quantize_weight(p, (int)a.x.type, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_rms_norm(const ftb_rms_norm_args* args, void* stream) {
  static const char fn[] = "ftb_rms_norm";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_rms_norm_args& a = *args;
    if (a.m == 0) return ST_OK;
    if (!a.x.data || (!a.y.data && !a.q.data) || (a.q.data && !a.q.scales)) return refuse(fn, "null pointer", ST_NULL);
    if (a.y.data && a.q.data) return refuse(fn, "y and q are both set");
    if (a.h.data && !a.residual.data) return refuse(fn, "h is the sum with a residual: pass one");
    if (!sizes_ok(a.m, 1, a.k)) return refuse(fn, "needs 0 <= m and 1 <= k, at most 2^27");
    if (!(a.eps >= 0.0)) return refuse(fn, "eps must not be negative");
    std::string why = check("x", a.x, a.k);
    const ftb_matrix* others[3] = {&a.residual, &a.h, &a.y};
    const char* names[3] = {"residual", "h", "y"};
    for (int i = 0; i < 3 && why.empty(); ++i) {
      if (!others[i]->data) continue;
      why = check(names[i], *others[i], a.k);
      if (why.empty() && others[i]->type != a.x.type) why = std::string(names[i]) + " must have x's type";
    }
    if (why.empty() && a.weight && !aligned(a.weight, 4)) why = "weight is not aligned to its type";
    if (why.empty() && a.q.data) why = check("q", a.q, a.k);
    const Span x = span(a.x, a.m, a.k), r = span(a.residual, a.m, a.k), h = span(a.h, a.m, a.k);
    const Span in[3] = {x, r, span(a.weight, 1, 4 * a.k, 0)};
    const Span more[4] = {x, r, in[2], h};
    if (why.empty()) why = clashes("h", h, in, &x, &r);
    if (why.empty() && a.y.data) why = clashes("y", span(a.y, a.m, a.k), in, &x, &r);
    if (why.empty() && a.y.data && overlap(span(a.y, a.m, a.k), h)) why = "y overlaps h";
    if (why.empty() && a.q.data) why = clashes("q", a.q, a.m, a.m, a.k, more);
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = a.x.data;
    p.x_ld = a.x.ld;
    p.residual = a.residual.data;
    p.r_ld = a.residual.ld;
    p.weight = a.weight;
    p.eps = (float)a.eps;
    p.h = a.h.data;
    p.h_ld = a.h.ld;
    p.y = a.y.data;
    p.y_ld = a.y.ld;
    p.q = a.q.data;
    p.q_ld = a.q.ld;
    p.s = a.q.scales;
    p.s_ld = a.q.scales_ld;
    p.m = a.m;
    p.k = a.k;
    return launched(fn, launch_rms_norm(p, (int)a.x.type, d->sm_count, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_fp8_linear(const ftb_fp8_linear_args* args, void* stream) {
  static const char fn[] = "ftb_fp8_linear";
  return guarded(fn, [&]() -> int {
    if (!args) return refuse(fn, "null arguments", ST_NULL);
    const ftb_fp8_linear_args& a = *args;
    if (a.m == 0) return ST_OK;
    if (!a.a.data || !a.a.scales || !a.w.data || !a.w.scales || (!a.y.data && !a.q.data) ||
        (a.q.data && !a.q.scales))
      return refuse(fn, "null pointer", ST_NULL);
    if (a.y.data && a.q.data) return refuse(fn, "y and q are both set");
    if (!sizes_ok(a.m, a.n, a.k)) return refuse(fn, "needs 0 <= m, 1 <= n and 1 <= k, at most 2^27");
    if (a.flags & ~(int64_t)FTB_FP8_RELU) return refuse(fn, "unknown flags");
    std::string why = check("a", a.a, a.k);
    if (why.empty()) why = check("w", a.w, a.k);
    if (why.empty() && a.bias && !aligned(a.bias, 4)) why = "bias is not aligned to its type";
    if (why.empty() && a.residual.data) why = check("residual", a.residual, a.n);
    if (why.empty() && a.y.data) why = check("y", a.y, a.n);
    if (why.empty() && a.q.data) why = check("q", a.q, a.n);
    const Span r = span(a.residual, a.m, a.n);
    const Span in[6] = {span(a.a.data, a.m, a.k, a.a.ld),
                        span(a.a.scales, a.m, fp8_blocks(a.k), a.a.scales_ld),
                        span(a.w.data, a.n, a.k, a.w.ld),
                        span(a.w.scales, fp8_blocks(a.n), fp8_blocks(a.k), a.w.scales_ld),
                        span(a.bias, 1, 4 * a.n, 0),
                        r};
    if (why.empty() && a.y.data)
      why = clashes("y", span(a.y, a.m, a.n), in, a.residual.type == a.y.type ? &r : nullptr);
    if (why.empty() && a.q.data) why = clashes("q", a.q, a.m, a.m, a.n, in);
    if (!why.empty()) return refuse(fn, why);
    OpDevice* d = nullptr;
    if (const int rc = op_device(fn, &d)) return rc;
    Fp8Operands o{a.a.data, a.a.ld, a.w.data, a.w.ld};
    Fp8Params p{};
    p.M = (int)a.m;
    p.N = (int)a.n;
    p.K = (int)a.k;
    p.sa = a.a.scales;
    p.sa_ld = a.a.scales_ld;
    p.sw = a.w.scales;
    p.sw_ld = a.w.scales_ld;
    p.e.bias = a.bias;
    p.e.residual = a.residual.data;
    p.e.res_ld = a.residual.ld;
    p.e.res_type = (int)a.residual.type;
    p.e.relu = (a.flags & FTB_FP8_RELU) != 0;
    p.e.y = a.q.data ? a.q.data : a.y.data;
    p.e.y_ld = a.q.data ? a.q.ld : a.y.ld;
    p.e.y_type = a.q.data ? kFp8Type : (int)a.y.type;
    p.e.ys = a.q.scales;
    p.e.ys_ld = a.q.scales_ld;
    p.e.res_vec = rows_aligned(a.residual);
    p.e.y_vec = rows_aligned(a.y);
    p.err = d->fault_dev;
    p.stall_test = op_stall();
    return launched(fn, launch_fp8_linear(o, p, *d, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_fp8_set_fault_injection(int stall) {
  g_fp8_stall.store(stall ? 1 : 0);
  return ST_OK;
}

FTB_API int ftb_fp8_set_kernel(int nt, int split) {
  if (nt == -1) {
    g_fp8_kernel.store(-1);
    return ST_OK;
  }
  const bool tile = (nt == 16 || nt == 32 || nt == 64 || nt == 128) &&
                    (split == 1 || split == 2 || split == 4 || split == 8);
  if (!tile && !(nt == 0 && split == 1))
    return refuse("ftb_fp8_set_kernel", "needs nt 16, 32, 64 or 128 with split 1, 2, 4 or 8, nt 0 with split 1, or nt -1");
  g_fp8_kernel.store(16 * nt + split);
  return ST_OK;
}
