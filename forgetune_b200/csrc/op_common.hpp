// What the entry points of the operators on device buffers share: the state of
// each device, argument checks and refusals.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <exception>
#include <mutex>
#include <string>

#include "forgetune_b200.h"
#include "status.hpp"

namespace ftb {

struct OpDevice {
  std::mutex mu;
  std::atomic<bool> ready{false};
  int sm_count = 0;
  int pairs = 0;  // SM pairs resident at once
  // set by a kernel whose bounded wait gave up: mapped host memory, so the
  // next call reads it without a copy
  volatile int* fault = nullptr;
  int* fault_dev = nullptr;
};

// The current device's state, set up by the first call on it (a set-up that
// fails is tried again by the next); refuses where an earlier kernel on the
// device gave up a wait (fp8.cu).
int op_device(const char* fn, OpDevice** out);

// Kernel attributes of the operators in decoder.cu, once per device.
cudaError_t decoder_prepare();

// Failure-detection hook: whether launches stall (ftb_fp8_set_fault_injection).
int op_stall();

inline int refuse(const char* fn, const std::string& why, int status = ST_INPUT) {
  set_error(std::string(fn) + ": " + why);
  return status;
}

inline bool is_plain(int64_t type) { return type == FTB_F32 || type == FTB_F16 || type == FTB_BF16; }
inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows of `cols` elements `ld` apart: enough room, and the alignment of the
// element type (plain) or of the copy engine (quantised).  "" when fine.
inline std::string check(const char* what, const ftb_matrix& x, int64_t cols) {
  if (!is_plain(x.type)) return std::string(what) + " must be float32, float16 or bfloat16";
  if (!aligned(x.data, x.type == FTB_F32 ? 4 : 2)) return std::string(what) + " is not aligned to its type";
  if (x.ld < cols) return std::string(what) + " rows overlap (stride below the row length)";
  return "";
}
// Base and rows on 16-byte boundaries.
inline bool rows_aligned(const ftb_matrix& x) {
  return aligned(x.data, 16) && (x.ld * (x.type == FTB_F32 ? 4 : 2)) % 16 == 0;
}
// Bytes of a matrix in memory: rows `ld` bytes apart.
struct Span {
  const char* p;
  int64_t rows, bytes, ld;
  int64_t end() const { return (rows - 1) * ld + bytes; }
};
inline Span span(const ftb_matrix& x, int64_t m, int64_t n) {
  const int64_t size = x.type == FTB_F32 ? 4 : 2;
  return {static_cast<const char*>(x.data), m, n * size, x.ld * size};
}
inline Span span(const void* p, int64_t rows, int64_t bytes, int64_t ld) {
  return {static_cast<const char*>(p), rows, bytes, ld};
}
inline bool overlap(const Span& a, const Span& b) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.p + a.end() <= b.p || b.p + b.end() <= a.p) return false;
  if (a.rows == 1 && b.rows == 1) return true;  // their ranges meet (a vector's span has no stride)
  const int64_t ld = a.rows > 1 ? a.ld : b.ld;
  if ((a.rows > 1 && a.ld != ld) || (b.rows > 1 && b.ld != ld)) return true;  // not worth telling apart
  const int64_t d = ((b.p - a.p) % ld + ld) % ld;  // b's columns in a's rows
  return !(d >= a.bytes && d + b.bytes <= ld);
}
inline bool same(const Span& a, const Span& b) {
  return a.p == b.p && a.rows == b.rows && a.bytes == b.bytes && (a.rows <= 1 || a.ld == b.ld);
}
// An output that shares memory with an operand, unless it is that operand in
// place: "" or why not.
template <size_t N>
inline std::string clashes(const char* what, const Span& out, const Span (&in)[N], const Span* in_place = nullptr,
                           const Span* in_place2 = nullptr) {
  for (const Span& x : in)
    if (overlap(out, x) && !(in_place && same(out, x) && same(*in_place, x)) &&
        !(in_place2 && same(out, x) && same(*in_place2, x)))
      return std::string(what) + " overlaps an operand";
  return "";
}

inline int launched(const char* fn, cudaError_t e) {
  if (e == cudaSuccess) return ST_OK;
  cudaGetLastError();
  return refuse(fn, std::string("launch failed: ") + cudaGetErrorString(e), ST_DEVICE);
}

template <typename F>
inline int guarded(const char* fn, F&& body) noexcept {
  try {
    return body();
  } catch (const std::exception& e) {
    try {
      return refuse(fn, e.what(), ST_ALLOC);
    } catch (...) {
      return ST_ALLOC;
    }
  } catch (...) {
    return ST_ALLOC;
  }
}

}  // namespace ftb
