// RMS norm of fp32 rows for the compiled graph's RMSNORM step (fp8.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace ftb {

// y = x / sqrt(mean(x^2) + eps) * weight over the rows of x [m, k]; weight may
// be null, y may be x.  Enqueued on `s`.
cudaError_t rms_norm_f32(const float* x, const float* weight, float eps, float* y, int64_t m, int64_t k, int sm_count,
                         cudaStream_t s);

}  // namespace ftb
