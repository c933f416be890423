// Kernels over rows: quantisation of activations and weights, and RMS norm
// with the residual's addition and a plain or quantised output.  All are
// bound by the bytes of their operands; each element is read and written once
// (rows too long for registers are read twice).
//
// A lane has a vector of VEC consecutive elements, 16 bytes of input: 8 of a
// 16-bit type, 4 of fp32.  A quantisation block of 128 is then 16 or 32
// neighbouring lanes, so its largest value is a few shuffles away.  Rows whose
// base, stride or length keep them off 16-byte boundaries take the same
// kernels with element-wise loads and stores (VECTOR false).
#pragma once

#include <algorithm>

#include "fp8_format.cuh"
#include "tc_ptx.cuh"

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

template <typename T>
constexpr int kRowVec = 16 / (int)sizeof(T);

// 16 bytes of T as fp32.
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x);
  v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z);
  v[3] = __uint_as_float(u.w);
}
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[8]);
template <>
__device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack16<__half>(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&v)[VEC]) {
  if constexpr (VEC == 4) unpack(u, v);
  else unpack16<T>(u, v);
}

template <typename T, int VEC>
__device__ __forceinline__ uint4 pack_vec(const float (&v)[VEC]) {
  T t[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) t[i] = from_f32<T>(v[i]);
  uint4 u;
  memcpy(&u, t, 16);
  return u;
}

// A lane's vector at column c: zeros past k.
template <typename T, bool VECTOR>
__device__ __forceinline__ uint4 load_vec(const T* row, int64_t c, int64_t k) {
  constexpr int VEC = kRowVec<T>;
  uint4 u = make_uint4(0, 0, 0, 0);
  if constexpr (VECTOR) {
    if (c < k) u = *reinterpret_cast<const uint4*>(row + c);
  } else {
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = c + i < k ? row[c + i] : from_f32<T>(0.0f);
    memcpy(&u, t, 16);
  }
  return u;
}

template <typename T, bool VECTOR>
__device__ __forceinline__ void store_vec(T* row, int64_t c, int64_t k, const float (&v)[kRowVec<T>]) {
  if constexpr (VECTOR) {
    if (c < k) *reinterpret_cast<uint4*>(row + c) = pack_vec<T>(v);
  } else {
#pragma unroll
    for (int i = 0; i < kRowVec<T>; ++i)
      if (c + i < k) row[c + i] = from_f32<T>(v[i]);
  }
}

// The largest of the block's 128 / VEC lanes.
template <int VEC>
__device__ __forceinline__ uint32_t block_max(uint32_t a) {
  if constexpr (VEC == 4) return __reduce_max_sync(0xffffffffu, a);
#pragma unroll
  for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// A warp quantises its lanes' vectors (VEC 8: two blocks, VEC 4: one) and
// stores values and scales; every lane takes part, also past k.
template <int VEC>
__device__ __forceinline__ void quantize_vec(float (&v)[VEC], uint8_t* qrow, uint8_t* srow, int64_t c, int64_t k) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  a = block_max<VEC>(a);
  if (__any_sync(0xffffffffu, a >= 0x7F800000u)) {
    // some value is not finite: the scale comes from the others
    a = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a = max(a, finite_abs_bits(v[i]));
      v[i] = nan_unless_finite(v[i]);
    }
    a = block_max<VEC>(a);
  }
  const uint32_t byte = fp8_scale_byte(a);
  const float inv = fp8_inv_scale(byte);
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) w[i] = fp8_pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  if (c + VEC <= k) {
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(qrow + c) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(qrow + c) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (c + i < k) qrow[c + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
  if (c % kFp8Block == 0 && c < k) srow[c / kFp8Block] = (uint8_t)byte;
}

// One warp per chunk of kQuantUnits x 32 vectors of a row, its loads issued
// together.
constexpr int kQuantUnits = 4;

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const RowsParams p, const uint32_t chunks) {
  constexpr int VEC = kRowVec<T>;
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t warp = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row = (warp >> 32) == 0 ? (int64_t)((uint32_t)warp / chunks) : warp / chunks;
  if (row >= p.m) return;
  const int64_t c0 = ((warp - row * chunks) * kQuantUnits * 32 + (threadIdx.x & 31)) * VEC;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  uint4 u[kQuantUnits];
#pragma unroll
  for (int j = 0; j < kQuantUnits; ++j) u[j] = load_vec<T, VECTOR>(x, c0 + j * 32 * VEC, p.k);
#pragma unroll
  for (int j = 0; j < kQuantUnits; ++j) {
    const int64_t c = c0 + j * 32 * VEC;
    float v[VEC];
    unpack_vec<T>(u[j], v);
    quantize_vec<VEC>(v, p.q + row * p.q_ld, p.s + row * p.s_ld, c, p.k);
  }
}

// One CTA per 128 x 128 block of a weight: the block's largest value first,
// then its values again.  Runs once per weight.
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(RowsParams p) {
  __shared__ uint32_t amax[8];
  grid_dep_wait();
  grid_dep_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * kFp8Block + lane * 4, r0 = (int64_t)blockIdx.y * kFp8Block;
  const T* x = static_cast<const T*>(p.x);
  uint32_t a = 0;
  for (int i = warp; i < kFp8Block && r0 + i < p.m; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < p.k) a = max(a, finite_abs_bits(to_f32(x[(r0 + i) * p.x_ld + c + j])));
  }
  a = __reduce_max_sync(0xffffffffu, a);
  if (lane == 0) amax[warp] = a;
  __syncthreads();
  a = __reduce_max_sync(0xffffffffu, amax[lane & 7]);
  const uint32_t byte = fp8_scale_byte(a);
  const float inv = fp8_inv_scale(byte);
  for (int i = warp; i < kFp8Block && r0 + i < p.m; i += 8) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = c + j < p.k ? nan_unless_finite(to_f32(x[(r0 + i) * p.x_ld + c + j])) : 0.0f;
    const uint32_t w = fp8_pack4(v[0], v[1], v[2], v[3], inv);
    uint8_t* q = p.q + (r0 + i) * p.q_ld;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < p.k) q[c + j] = (uint8_t)(w >> (8 * j));
  }
  if (threadIdx.x == 0) p.s[blockIdx.y * p.s_ld + blockIdx.x] = (uint8_t)byte;
}

// Sum of the squares, pairwise.
template <int VEC>
__device__ __forceinline__ float square_sum(const float (&v)[VEC]) {
  float t[VEC / 2];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) t[i] = v[2 * i] * v[2 * i] + v[2 * i + 1] * v[2 * i + 1];
#pragma unroll
  for (int n = VEC / 4; n; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) t[i] += t[i + n];
  return t[0];
}

// What follows once a vector's h and its row's scale are known.
template <typename T, bool VECTOR>
__device__ __forceinline__ void norm_finish(const RowsParams& p, int64_t row, int64_t c, float scale,
                                            float (&v)[kRowVec<T>]) {
  constexpr int VEC = kRowVec<T>;
  if (p.h) store_vec<T, VECTOR>(static_cast<T*>(p.h) + row * p.h_ld, c, p.k, v);
  if (p.weight) {
    if (VECTOR && c < p.k) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 w = *reinterpret_cast<const float4*>(p.weight + c + i);
        v[i] = v[i] * scale * w.x;
        v[i + 1] = v[i + 1] * scale * w.y;
        v[i + 2] = v[i + 2] * scale * w.z;
        v[i + 3] = v[i + 3] * scale * w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = c + i < p.k ? v[i] * scale * p.weight[c + i] : 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= scale;
  }
  if (p.q) quantize_vec<VEC>(v, p.q + row * p.q_ld, p.s + row * p.s_ld, c, p.k);
  else store_vec<T, VECTOR>(static_cast<T*>(p.y) + row * p.y_ld, c, p.k, v);
}

//   h = x + residual (fp32),  y = h / sqrt(mean(h^2) + eps) weight
// `warps` warps per row, which keep it in registers: NV vectors per lane.  A
// CTA has one row, or several short ones.
template <typename T, bool VECTOR, int NV>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const RowsParams p, const int warps) {
  constexpr int VEC = kRowVec<T>;
  __shared__ float part[32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = w / warps * warps;  // the first warp of this one's row
  const int64_t row = (int64_t)blockIdx.x * ((blockDim.x >> 5) / warps) + w / warps;
  const int64_t c0 = (int64_t)((w - first) * 32 + lane) * VEC, step = (int64_t)warps * 32 * VEC;
  grid_dep_wait();
  grid_dep_trigger();
  float v[NV][VEC];
  float ss = 0.0f;
  if (row < p.m) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* r = static_cast<const T*>(p.residual) + row * p.r_ld;
    uint4 xu[NV], ru[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) xu[j] = load_vec<T, VECTOR>(x, c0 + j * step, p.k);
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < NV; ++j) ru[j] = load_vec<T, VECTOR>(r, c0 + j * step, p.k);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack_vec<T>(xu[j], v[j]);
      if (p.residual) {
        float t[VEC];
        unpack_vec<T>(ru[j], t);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] += t[i];
      }
      ss += square_sum(v[j]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (warps > 1) {
    if (lane == 0) part[w] = ss;
    __syncthreads();
    ss = lane < warps ? part[first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  if (row >= p.m) return;
  const float scale = rsqrtf(ss / (float)p.k + p.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) norm_finish<T, VECTOR>(p, row, c0 + j * step, scale, v[j]);
}

// Rows too long for registers: one CTA per row, which reads it twice.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const RowsParams p) {
  constexpr int VEC = kRowVec<T>;
  __shared__ float part[32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.r_ld : nullptr;
  const int64_t step = 1024 * VEC;
  auto load = [&](int64_t c, float (&v)[VEC]) {
    unpack_vec<T>(load_vec<T, VECTOR>(x, c, p.k), v);
    if (r) {
      float t[VEC];
      unpack_vec<T>(load_vec<T, VECTOR>(r, c, p.k), t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] += t[i];
    }
  };
  float ss = 0.0f;
  for (int64_t c = (int64_t)threadIdx.x * VEC; c < p.k; c += step) {
    float v[VEC];
    load(c, v);
    ss += square_sum(v);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[w] = ss;
  __syncthreads();
  ss = part[lane];
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float scale = rsqrtf(ss / (float)p.k + p.eps);
  for (int64_t c0 = (int64_t)w * 32 * VEC; c0 < p.k; c0 += step) {  // whole warps: they quantise together
    float v[VEC];
    load(c0 + lane * VEC, v);
    norm_finish<T, VECTOR>(p, row, c0 + lane * VEC, scale, v);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Rows that vectors of 16 bytes cover exactly.
template <typename T>
inline bool rows_vector(const void* p, int64_t ld, int64_t rows) {
  return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows <= 1 || ld % kRowVec<T> == 0));
}

template <typename T>
inline cudaError_t launch_quantize_rows_t(const RowsParams& p, cudaStream_t s) {
  const int64_t chunk = kQuantUnits * 32 * kRowVec<T>;
  const int64_t chunks = (p.k + chunk - 1) / chunk;
  const int64_t grid = (p.m * chunks + 7) / 8;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const bool vec = p.k % kRowVec<T> == 0 && rows_vector<T>(p.x, p.x_ld, p.m);
  return pdl_launch(vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, dim3((unsigned)grid),
                    dim3(256), 0, s, p, (uint32_t)chunks);
}
inline cudaError_t launch_quantize_rows(const RowsParams& p, int type, cudaStream_t s) {
  if (type == FTB_F32) return launch_quantize_rows_t<float>(p, s);
  if (type == FTB_F16) return launch_quantize_rows_t<__half>(p, s);
  return launch_quantize_rows_t<__nv_bfloat16>(p, s);
}

inline cudaError_t launch_quantize_weight(const RowsParams& p, int type, cudaStream_t s) {
  const dim3 grid((unsigned)fp8_blocks(p.k), (unsigned)fp8_blocks(p.m));
  return pdl_launch(type == FTB_F32   ? quantize_weight_kernel<float>
                    : type == FTB_F16 ? quantize_weight_kernel<__half>
                                      : quantize_weight_kernel<__nv_bfloat16>,
                    grid, dim3(256), 0, s, p);
}

template <typename T, bool VECTOR>
inline cudaError_t launch_rms_norm_v(const RowsParams& p, int sm_count, cudaStream_t s) {
  const int64_t vectors = (p.k + kRowVec<T> - 1) / kRowVec<T>;
  constexpr int64_t kMost = 1024 * 4;  // vectors of a row that the registers of 1024 threads hold
  if (vectors > kMost)
    return pdl_launch(rms_norm_long_kernel<T, VECTOR>, dim3((unsigned)p.m), dim3(1024), 0, s, p);
  // Many rows: four vectors per lane, so that few warps share a row and many
  // loads are in flight.  Few rows: one per lane, the shortest time.
  const int nv = p.m >= 2 * sm_count || vectors > 1024 ? 4 : 1;
  int warps = 1;
  while (warps * 32 * nv < vectors) warps *= 2;
  const int rows = std::max(1, 8 / warps);
  const unsigned grid = (unsigned)((p.m + rows - 1) / rows);
  return pdl_launch(nv == 4 ? rms_norm_kernel<T, VECTOR, 4> : rms_norm_kernel<T, VECTOR, 1>, dim3(grid),
                    dim3(32 * warps * rows), 0, s, p, warps);
}
template <typename T>
inline cudaError_t launch_rms_norm_t(const RowsParams& p, int sm_count, cudaStream_t s) {
  const bool vec = p.k % kRowVec<T> == 0 && rows_vector<T>(p.x, p.x_ld, p.m) &&
                   rows_vector<T>(p.residual, p.r_ld, p.m) && rows_vector<T>(p.h, p.h_ld, p.m) &&
                   rows_vector<T>(p.y, p.y_ld, p.m) && (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0;
  return vec ? launch_rms_norm_v<T, true>(p, sm_count, s) : launch_rms_norm_v<T, false>(p, sm_count, s);
}
inline cudaError_t launch_rms_norm(const RowsParams& p, int type, int sm_count, cudaStream_t s) {
  if (type == FTB_F32) return launch_rms_norm_t<float>(p, sm_count, s);
  if (type == FTB_F16) return launch_rms_norm_t<__half>(p, sm_count, s);
  return launch_rms_norm_t<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace ftb
