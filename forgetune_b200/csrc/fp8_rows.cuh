// Kernels over rows: quantisation of activations and weights, and RMS norm
// with the residual's addition and a plain or quantised output.
#pragma once

#include <algorithm>

#include "fp8_format.cuh"

namespace ftb {

struct RowsParams {
  const void* x;
  int64_t x_ld;
  const void* residual;  // added to x (norm only), or null
  int64_t r_ld;
  const float* weight;  // norm only, or null
  float eps;
  void* h;  // x + residual in x's type, or null
  int64_t h_ld;
  void* y;  // plain output in x's type, or null
  int64_t y_ld;
  uint8_t* q;  // quantised output, or null
  int64_t q_ld;
  uint8_t* s;
  int64_t s_ld;
  int64_t m, k;
};

// Lane l's four values of a block: elements 4 l .. 4 l + 3, zero past `k`.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int64_t c, int64_t k, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = c + i < k ? to_f32(row[c + i]) : 0.0f;
}

// A warp quantises one block from its lanes' four values each.
__device__ __forceinline__ void quantize_block(const float (&v)[4], uint8_t* qrow, uint8_t* s, int64_t c, int64_t k,
                                               int lane) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, finite_abs_bits(v[i]));
  const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, a));
  const uint32_t w = fp8_pack4(v[0], v[1], v[2], v[3], fp8_inv_scale(byte));
  if (c + 3 < k) {
    *reinterpret_cast<uint32_t*>(qrow + c) = w;
  } else {
    for (int i = 0; i < 4; ++i)
      if (c + i < k) qrow[c + i] = (uint8_t)(w >> (8 * i));
  }
  if (lane == 0) *s = (uint8_t)byte;
}

// One warp per block of 128 of a row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(RowsParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t kb = (p.k + kFp8Block - 1) / kFp8Block;
  const int64_t units = p.m * kb, step = (int64_t)gridDim.x * 8;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t row = u / kb, b = u - row * kb, c = b * kFp8Block + lane * 4;
    float v[4];
    load4(static_cast<const T*>(p.x) + row * p.x_ld, c, p.k, v);
    quantize_block(v, p.q + row * p.q_ld, p.s + row * p.s_ld + b, c, p.k, lane);
  }
}

// One CTA per 128 x 128 block of a weight: the block's largest value first,
// then its values again.
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(RowsParams p) {
  __shared__ uint32_t amax[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * kFp8Block + lane * 4, r0 = (int64_t)blockIdx.y * kFp8Block;
  const T* x = static_cast<const T*>(p.x);
  uint32_t a = 0;
  float v[4];
  for (int i = warp; i < kFp8Block && r0 + i < p.m; i += 8) {
    load4(x + (r0 + i) * p.x_ld, c, p.k, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, finite_abs_bits(v[j]));
  }
  a = __reduce_max_sync(0xffffffffu, a);
  if (lane == 0) amax[warp] = a;
  __syncthreads();
  a = __reduce_max_sync(0xffffffffu, amax[lane & 7]);
  const uint32_t byte = fp8_scale_byte(a);
  const float inv = fp8_inv_scale(byte);
  for (int i = warp; i < kFp8Block && r0 + i < p.m; i += 8) {
    load4(x + (r0 + i) * p.x_ld, c, p.k, v);
    const uint32_t w = fp8_pack4(v[0], v[1], v[2], v[3], inv);
    uint8_t* q = p.q + (r0 + i) * p.q_ld;
    for (int j = 0; j < 4; ++j)
      if (c + j < p.k) q[c + j] = (uint8_t)(w >> (8 * j));
  }
  if (threadIdx.x == 0) p.s[blockIdx.y * p.s_ld + blockIdx.x] = (uint8_t)byte;
}

// One CTA per row; the second pass reads the row again.
//   h = x + residual (fp32),  y = h / sqrt(mean(h^2) + eps) weight
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_kernel(RowsParams p) {
  __shared__ float part[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t row = blockIdx.x; row < p.m; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.r_ld : nullptr;
    float ss = 0.0f;
    for (int64_t c = warp * kFp8Block + lane * 4; c < p.k; c += 8 * kFp8Block) {
      float v[4], w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      load4(x, c, p.k, v);
      if (r) load4(r, c, p.k, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += (v[i] + w[i]) * (v[i] + w[i]);
    }
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int i = 0; i < 8; ++i) ss += part[i];
    __syncthreads();
    const float scale = rsqrtf(ss / (float)p.k + p.eps);
    for (int64_t c0 = warp * kFp8Block; c0 < p.k; c0 += 8 * kFp8Block) {
      const int64_t c = c0 + lane * 4;
      float v[4], w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      load4(x, c, p.k, v);
      if (r) load4(r, c, p.k, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] += w[i];
        if (p.h && c + i < p.k) (static_cast<T*>(p.h) + row * p.h_ld)[c + i] = from_f32<T>(v[i]);
        v[i] = v[i] * scale * (p.weight && c + i < p.k ? p.weight[c + i] : 1.0f);
        if (p.y && c + i < p.k) (static_cast<T*>(p.y) + row * p.y_ld)[c + i] = from_f32<T>(v[i]);
      }
      if (p.q) quantize_block(v, p.q + row * p.q_ld, p.s + row * p.s_ld + c0 / kFp8Block, c, p.k, lane);
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T>
inline cudaError_t launch_quantize_rows_t(const RowsParams& p, int sm_count, cudaStream_t s) {
  const int64_t units = p.m * fp8_blocks(p.k);
  const unsigned grid = (unsigned)std::min<int64_t>((units + 7) / 8, (int64_t)sm_count * 16);
  quantize_rows_kernel<T><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}
inline cudaError_t launch_quantize_rows(const RowsParams& p, int type, int sm_count, cudaStream_t s) {
  if (type == FTB_F32) return launch_quantize_rows_t<float>(p, sm_count, s);
  if (type == FTB_F16) return launch_quantize_rows_t<__half>(p, sm_count, s);
  return launch_quantize_rows_t<__nv_bfloat16>(p, sm_count, s);
}

inline cudaError_t launch_quantize_weight(const RowsParams& p, int type, cudaStream_t s) {
  const int64_t rows = fp8_blocks(p.m);
  if (rows > 65535) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)fp8_blocks(p.k), (unsigned)rows);
  if (type == FTB_F32) quantize_weight_kernel<float><<<grid, 256, 0, s>>>(p);
  else if (type == FTB_F16) quantize_weight_kernel<__half><<<grid, 256, 0, s>>>(p);
  else quantize_weight_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
inline cudaError_t launch_rms_norm_t(const RowsParams& p, int sm_count, cudaStream_t s) {
  const unsigned grid = (unsigned)std::min<int64_t>(p.m, (int64_t)sm_count * 32);
  rms_norm_kernel<T><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}
inline cudaError_t launch_rms_norm(const RowsParams& p, int type, int sm_count, cudaStream_t s) {
  if (type == FTB_F32) return launch_rms_norm_t<float>(p, sm_count, s);
  if (type == FTB_F16) return launch_rms_norm_t<__half>(p, sm_count, s);
  return launch_rms_norm_t<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace ftb
