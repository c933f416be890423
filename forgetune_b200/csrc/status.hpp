// Status codes of the C ABI and the calling thread's error message.
#pragma once

#include <string>

namespace ftb {

// include/forgetune_b200.h
enum Status : int {
  ST_OK = 0,
  ST_NULL = -1,
  ST_INPUT = -2,
  ST_OUTPUT = -3,
  ST_ALLOC = -4,
  ST_DEVICE = -5,
  ST_CONFIG = -6,
};

// Keeps `s` for ftb_last_error() on this thread (runtime.cu).
void set_error(const std::string& s);

}  // namespace ftb

#define FTB_API extern "C" __attribute__((visibility("default")))

#define CUDA_TRY(expr)                                                                 \
  do {                                                                                 \
    cudaError_t _e = (expr);                                                           \
    if (_e != cudaSuccess) {                                                           \
      ftb::set_error(std::string(#expr) + ": " + cudaGetErrorString(_e));             \
      return ftb::ST_DEVICE;                                                           \
    }                                                                                  \
  } while (0)
