// C entry points of the block-scaled 8-bit operators
// (include/forgetune_b200.h): argument checks, the per-device set-up and the
// launches.
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>
#include <string>

#include "forgetune_b200.h"
#include "fp8_gemm.cuh"
#include "fp8_rows.cuh"
#include "status.hpp"

namespace ftb {

constexpr int kFp8MaxDevices = 64;
constexpr int64_t kFp8MaxDim = int64_t(1) << 30;

struct Fp8Device {
  std::once_flag once;
  int rc = ST_OK;
  std::string err;
  int sm_count = 0;
  // set by a kernel whose bounded wait gave up: mapped host memory, so the
  // next call reads it without a copy
  volatile int* fault = nullptr;
  int* fault_dev = nullptr;
};
static Fp8Device g_fp8_devices[kFp8MaxDevices];

static int refuse(const char* fn, const std::string& why, int status = ST_INPUT) {
  set_error(std::string(fn) + ": " + why);
  return status;
}

static void fp8_setup(int dev, Fp8Device* d) {
  cudaError_t e = cudaDeviceGetAttribute(&d->sm_count, cudaDevAttrMultiProcessorCount, dev);
  int major = 0;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess && major != 10) {
    d->rc = ST_DEVICE;
    d->err = "needs a GPU of compute capability 10.0 (sm_100a)";
    return;
  }
  void* h = nullptr;
  if (e == cudaSuccess) e = cudaHostAlloc(&h, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
  void* hd = nullptr;
  if (e == cudaSuccess) {
    *static_cast<int*>(h) = 0;
    e = cudaHostGetDevicePointer(&hd, h, 0);
  }
  if (e == cudaSuccess) e = fp8_tile_attributes<16>();
  if (e == cudaSuccess) e = fp8_tile_attributes<32>();
  if (e == cudaSuccess) e = fp8_tile_attributes<64>();
  if (e == cudaSuccess) e = fp8_tile_attributes<128>();
  if (e != cudaSuccess) {
    d->rc = ST_DEVICE;
    d->err = std::string("set-up failed: ") + cudaGetErrorString(e);
    cudaGetLastError();
    return;
  }
  d->fault = static_cast<volatile int*>(h);
  d->fault_dev = static_cast<int*>(hd);
}

// The current device's state, set up by the first call on it.
static int fp8_device(const char* fn, Fp8Device** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return refuse(fn, cudaGetErrorString(e), ST_DEVICE);
  }
  if (dev < 0 || dev >= kFp8MaxDevices) return refuse(fn, "device ordinal beyond the supported range", ST_CONFIG);
  Fp8Device& d = g_fp8_devices[dev];
  std::call_once(d.once, [&]() { fp8_setup(dev, &d); });
  if (d.rc != ST_OK) return refuse(fn, d.err, d.rc);
  const int code = *d.fault;
  if (code != 0) {
    *d.fault = 0;
    return refuse(fn, "an earlier call on this device gave up a wait (code " + std::to_string(code) +
                          "); its output is not valid", ST_DEVICE);
  }
  *out = &d;
  return ST_OK;
}

static bool is_plain(int type) { return type == FTB_F32 || type == FTB_F16 || type == FTB_BF16; }
static bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
static int64_t type_size(int type) { return type == FTB_F32 ? 4 : type == FTB_E4M3 ? 1 : 2; }

// Rows of `cols` elements `ld` apart: enough room, and the alignment of the
// element type (plain) or of the copy engine (quantised).  "" when fine.
static std::string check_plain(const char* what, const void* p, int type, int64_t cols, int64_t ld) {
  if (!aligned(p, (uintptr_t)type_size(type))) return std::string(what) + " is not aligned to its type";
  if (ld < cols) return std::string(what) + " rows overlap (stride below the row length)";
  return "";
}
static std::string check_quantized(const char* what, const void* q, int64_t q_ld, const void* s, int64_t s_ld,
                                   int64_t cols) {
  if (!aligned(q, 16) || q_ld % 16 || q_ld < cols)
    return std::string(what) + " values need 16-byte aligned rows (base and stride) of at least their length";
  if (!aligned(s, 4) || s_ld % 4 || s_ld < fp8_blocks(cols))
    return std::string(what) + " scales need 4-byte aligned rows (base and stride) of at least their length";
  return "";
}

static int launched(const char* fn, cudaError_t e) {
  if (e == cudaSuccess) return ST_OK;
  cudaGetLastError();
  return refuse(fn, std::string("launch failed: ") + cudaGetErrorString(e), ST_DEVICE);
}

template <typename F>
static int guarded(const char* fn, F&& body) noexcept {
  try {
    return body();
  } catch (const std::exception& e) {
    try {
      return refuse(fn, e.what(), ST_ALLOC);
    } catch (...) {
      return ST_ALLOC;
    }
  }
}

}  // namespace ftb

using namespace ftb;

FTB_API int ftb_quantize_rows(const void* x, int x_type, int64_t x_ld, uint8_t* q, int64_t q_ld, uint8_t* scales,
                              int64_t s_ld, int64_t m, int64_t k, void* stream) {
  static const char fn[] = "ftb_quantize_rows";
  return guarded(fn, [&]() -> int {
    if (m == 0) return ST_OK;
    if (!x || !q || !scales) return refuse(fn, "null pointer", ST_NULL);
    if (m < 0 || m > kFp8MaxDim || k < 1 || k > kFp8MaxDim) return refuse(fn, "needs 0 <= m and 1 <= k, at most 2^30");
    if (!is_plain(x_type)) return refuse(fn, "x is float32, float16 or bfloat16");
    std::string why = check_plain("x", x, x_type, k, x_ld);
    if (why.empty()) why = check_quantized("output", q, q_ld, scales, s_ld, k);
    if (!why.empty()) return refuse(fn, why);
    Fp8Device* d = nullptr;
    if (const int rc = fp8_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = x;
    p.x_ld = x_ld;
    p.q = q;
    p.q_ld = q_ld;
    p.s = scales;
    p.s_ld = s_ld;
    p.m = m;
    p.k = k;
    return launched(fn, launch_quantize_rows(p, x_type, d->sm_count, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_quantize_weight(const void* w, int w_type, int64_t w_ld, uint8_t* q, int64_t q_ld, uint8_t* scales,
                                int64_t s_ld, int64_t n, int64_t k, void* stream) {
  static const char fn[] = "ftb_quantize_weight";
  return guarded(fn, [&]() -> int {
    if (!w || !q || !scales) return refuse(fn, "null pointer", ST_NULL);
    if (n < 1 || n > kFp8MaxDim || k < 1 || k > kFp8MaxDim) return refuse(fn, "needs 1 <= n and 1 <= k, at most 2^30");
    if (!is_plain(w_type)) return refuse(fn, "w is float32, float16 or bfloat16");
    std::string why = check_plain("w", w, w_type, k, w_ld);
    if (why.empty()) why = check_quantized("output", q, q_ld, scales, s_ld, k);
    if (!why.empty()) return refuse(fn, why);
    Fp8Device* d = nullptr;
    if (const int rc = fp8_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = w;
    p.x_ld = w_ld;
    p.q = q;
    p.q_ld = q_ld;
    p.s = scales;
    p.s_ld = s_ld;
    p.m = n;
    p.k = k;
    return launched(fn, launch_quantize_weight(p, w_type, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_rms_norm(const void* x, int x_type, int64_t x_ld, const void* residual, int64_t r_ld,
                         const float* weight, float eps, void* h, int64_t h_ld, void* y, int y_type, int64_t y_ld,
                         uint8_t* scales, int64_t s_ld, int64_t m, int64_t k, void* stream) {
  static const char fn[] = "ftb_rms_norm";
  return guarded(fn, [&]() -> int {
    if (m == 0) return ST_OK;
    if (!x || !y || (y_type == FTB_E4M3 && !scales)) return refuse(fn, "null pointer", ST_NULL);
    if (h && !residual) return refuse(fn, "h is the sum with a residual: pass one");
    if (m < 0 || m > kFp8MaxDim || k < 1 || k > kFp8MaxDim) return refuse(fn, "needs 0 <= m and 1 <= k, at most 2^30");
    if (!is_plain(x_type)) return refuse(fn, "x is float32, float16 or bfloat16");
    if (y_type != x_type && y_type != FTB_E4M3) return refuse(fn, "y has x's type or is quantised");
    if (!(eps >= 0.0f)) return refuse(fn, "eps must not be negative");
    std::string why = check_plain("x", x, x_type, k, x_ld);
    if (why.empty() && residual) why = check_plain("residual", residual, x_type, k, r_ld);
    if (why.empty() && h) why = check_plain("h", h, x_type, k, h_ld);
    if (why.empty() && weight && !aligned(weight, 4)) why = "weight is not aligned to its type";
    if (why.empty())
      why = y_type == FTB_E4M3 ? check_quantized("output", y, y_ld, scales, s_ld, k)
                               : check_plain("y", y, y_type, k, y_ld);
    if (!why.empty()) return refuse(fn, why);
    Fp8Device* d = nullptr;
    if (const int rc = fp8_device(fn, &d)) return rc;
    RowsParams p{};
    p.x = x;
    p.x_ld = x_ld;
    p.residual = residual;
    p.r_ld = r_ld;
    p.weight = weight;
    p.eps = eps;
    p.h = h;
    p.h_ld = h_ld;
    if (y_type == FTB_E4M3) {
      p.q = static_cast<uint8_t*>(y);
      p.q_ld = y_ld;
      p.s = scales;
      p.s_ld = s_ld;
    } else {
      p.y = y;
      p.y_ld = y_ld;
    }
    p.m = m;
    p.k = k;
    return launched(fn, launch_rms_norm(p, x_type, d->sm_count, static_cast<cudaStream_t>(stream)));
  });
}

FTB_API int ftb_fp8_linear(const uint8_t* a, int64_t a_ld, const uint8_t* a_scales, int64_t as_ld, const uint8_t* w,
                           int64_t w_ld, const uint8_t* w_scales, int64_t ws_ld, const float* bias,
                           const void* residual, int r_type, int64_t r_ld, void* y, int y_type, int64_t y_ld,
                           uint8_t* y_scales, int64_t ys_ld, int64_t m, int64_t n, int64_t k, uint32_t flags,
                           void* stream) {
  static const char fn[] = "ftb_fp8_linear";
  return guarded(fn, [&]() -> int {
    if (m == 0) return ST_OK;
    if (!a || !a_scales || !w || !w_scales || !y || (y_type == FTB_E4M3 && !y_scales))
      return refuse(fn, "null pointer", ST_NULL);
    if (m < 0 || m > kFp8MaxDim || n < 1 || n > kFp8MaxDim || k < 1 || k > kFp8MaxDim)
      return refuse(fn, "needs 0 <= m, 1 <= n and 1 <= k, at most 2^30");
    if (flags & ~(uint32_t)FTB_FP8_RELU) return refuse(fn, "unknown flags");
    if (!is_plain(y_type) && y_type != FTB_E4M3) return refuse(fn, "y is float32, float16, bfloat16 or quantised");
    if (residual && !is_plain(r_type)) return refuse(fn, "residual is float32, float16 or bfloat16");
    std::string why = check_quantized("a", a, a_ld, a_scales, as_ld, k);
    if (why.empty()) why = check_quantized("w", w, w_ld, w_scales, ws_ld, k);
    if (why.empty() && bias && !aligned(bias, 4)) why = "bias is not aligned to its type";
    if (why.empty() && residual) why = check_plain("residual", residual, r_type, n, r_ld);
    if (why.empty())
      why = y_type == FTB_E4M3 ? check_quantized("output", y, y_ld, y_scales, ys_ld, n)
                               : check_plain("y", y, y_type, n, y_ld);
    if (!why.empty()) return refuse(fn, why);
    Fp8Device* d = nullptr;
    if (const int rc = fp8_device(fn, &d)) return rc;
    Fp8Operands o{a, a_ld, w, w_ld};
    Fp8Params p{};
    p.M = (int)m;
    p.N = (int)n;
    p.K = (int)k;
    p.sa = a_scales;
    p.sa_ld = as_ld;
    p.sw = w_scales;
    p.sw_ld = ws_ld;
    p.e.bias = bias;
    p.e.residual = residual;
    p.e.res_ld = r_ld;
    p.e.res_type = r_type;
    p.e.relu = (flags & FTB_FP8_RELU) != 0;
    p.e.y = y;
    p.e.y_ld = y_ld;
    p.e.y_type = y_type;
    p.e.ys = y_scales;
    p.e.ys_ld = ys_ld;
    p.err = d->fault_dev;
    return launched(fn, launch_fp8_linear(o, p, static_cast<cudaStream_t>(stream)));
  });
}
