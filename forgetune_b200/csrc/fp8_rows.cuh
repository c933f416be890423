// Kernels over rows: quantisation of activations and weights, and RMS norm
// with the residual's addition and a plain or quantised output.  All are
// bound by the bytes of their operands; each element is read and written once
// (rows too long for registers are read twice).
//
// A lane has a vector of VEC consecutive elements, 16 bytes of input: 8 of a
// 16-bit type, 4 of fp32.  A quantisation block of 128 is then 16 or 32
// neighbouring lanes, so its largest value is a few shuffles away.  Rows whose
// base, stride or length keep them off 16-byte boundaries are quantised by the
// same kernels with element-wise loads; the norm has kernels of its own for them
// (rms_norm_elements_kernel and a form of rms_norm_long_kernel).
#pragma once

#include <algorithm>
#include <cstring>
#include <type_traits>

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

// How a kernel's lanes meet its rows.
enum RowMode : int {
  ROW_ELEMENTS,  // element by element
  ROW_VECTORS,   // 16 bytes at a time; a lane's vector is inside the row or past its end
  ROW_WHOLE,     // and no lane's vector is past the end
};

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
template <typename T, RowMode MODE>
__device__ __forceinline__ uint4 load_vec(const T* row, int c, int k) {
  constexpr int VEC = kRowVec<T>;
  uint4 u = make_uint4(0, 0, 0, 0);
  if constexpr (MODE != ROW_ELEMENTS) {
    if (MODE == ROW_WHOLE || c < k) u = *reinterpret_cast<const uint4*>(row + c);
  } else {
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = c + i < k ? row[c + i] : from_f32<T>(0.0f);
    memcpy(&u, t, 16);
  }
  return u;
}

template <typename T, RowMode MODE>
__device__ __forceinline__ void store_vec(T* row, int c, int k, const float (&v)[kRowVec<T>]) {
  if (MODE == ROW_WHOLE || c < k) *reinterpret_cast<uint4*>(row + c) = pack_vec<T>(v);
}

// The scale byte plus one of a lane's largest |x| (as bits), 0 where all are
// zero, above 0xFF where one is not finite.  Adding 0x1FFFFF carries into the
// exponent exactly where the mantissa is above 1.75 (see fp8_scale_byte).
__device__ __forceinline__ uint32_t scale_code(uint32_t a) {
  const int b = (int)((a + 0x1FFFFFu) >> 23) - 7;
  const uint32_t c = (uint32_t)max(b, 1);
  return a == 0u ? 0u : a >= 0x7F800000u ? 0x1FFu : c;
}

// The largest of each block's 128 / VEC neighbouring lanes, of values below
// 2^16.  For VEC 8 two vectors share a word, which halves the shuffles.
template <int VEC, int N>
__device__ __forceinline__ void block_max16(uint32_t (&x)[N]) {
  if constexpr (VEC == 4) {
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = __reduce_max_sync(0xffffffffu, x[n]);
  } else {
    constexpr int W = (N + 1) / 2;
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = x[2 * i] | (2 * i + 1 < N ? x[(2 * i + 1) % N] << 16 : 0u);
#pragma unroll
    for (int o = 8; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = __vmaxu2(w[i], __shfl_xor_sync(0xffffffffu, w[i], o));
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = (n & 1) ? w[n / 2] >> 16 : w[n / 2] & 0xFFFFu;
  }
}

// Where a lane's vector goes: its place in the row's values and its block's
// place among the scales, and how many columns the row still has there.
struct VecPlace {
  uint8_t *q, *s;
  int left;
};

// One vector and, from the block's first lane, its scale.
template <bool WHOLE, int VEC>
__device__ __forceinline__ void store_quantized(const float (&v)[VEC], uint32_t byte, const VecPlace& o) {
  const float inv = fp8_inv_scale(byte);
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) w[i] = fp8_pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  if (WHOLE || o.left >= VEC) {
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(o.q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(o.q) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < o.left) o.q[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
  if ((threadIdx.x & (kFp8Block / VEC - 1)) == 0 && (WHOLE || o.left > 0)) *o.s = (uint8_t)byte;
}

// A warp quantises N vectors per lane at once (a vector's 32 lanes are two
// blocks for VEC 8, one for VEC 4) and stores values and scales where at(n)
// says.  Every lane takes part, also past the row's end.  `a`: the bits of
// each vector's largest |x|.  WHOLE: every vector is inside its row.
template <bool WHOLE, int VEC, int N, typename At>
__device__ __forceinline__ void quantize_vecs(float (&v)[N][VEC], const uint32_t (&a)[N], At&& at) {
  uint32_t code[N];
  uint32_t most = 0;
#pragma unroll
  for (int n = 0; n < N; ++n) code[n] = scale_code(a[n]), most = max(most, code[n]);
  if (__any_sync(0xffffffffu, most > 0xFFu)) {
    // some value is not finite: the scales come from the others
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t f = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        f = max(f, finite_abs_bits(v[n][i]));
        v[n][i] = nan_unless_finite(v[n][i]);
      }
      code[n] = scale_code(f);
    }
  }
  block_max16<VEC>(code);
#pragma unroll
  for (int n = 0; n < N; ++n) store_quantized<WHOLE>(v[n], code[n] ? code[n] - 1u : 127u, at(n));
}

// Bits of the largest |v|; NaN is passed over (it converts to NaN by itself).
template <int VEC>
__device__ __forceinline__ uint32_t abs_max_bits(const float (&v)[VEC]) {
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) a = fmaxf(a, fabsf(v[i]));
  return __float_as_uint(a);
}

// The same from 16 bytes of a 16-bit type, which compare two at a time as
// integers; the result is the 16 bits.
__device__ __forceinline__ uint32_t abs_max_bits16(const uint4& u) {
  const uint32_t m = 0x7FFF7FFFu;
  const uint32_t w = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  return max(w >> 16, w & 0xFFFFu);
}
// ... as the bits of fp32.
template <typename T>
__device__ __forceinline__ uint32_t widen_bits(uint32_t h) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

// A warp's N vectors as loaded, into values and scales.  A 16-bit type's
// largest values go through the shuffles as they are, two to a word.
template <typename T, bool WHOLE, int N, typename At>
__device__ __forceinline__ void quantize_loaded(const uint4 (&u)[N], At&& at) {
  constexpr int VEC = kRowVec<T>;
  float v[N][VEC];
#pragma unroll
  for (int n = 0; n < N; ++n) unpack_vec<T>(u[n], v[n]);
  if constexpr (VEC == 8) {
    constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
    uint32_t h[N], most = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) h[n] = abs_max_bits16(u[n]), most = max(most, h[n]);
    if (!__any_sync(0xffffffffu, most >= kInf)) {
      block_max16<VEC>(h);
#pragma unroll
      for (int n = 0; n < N; ++n)
        store_quantized<WHOLE>(v[n], fp8_scale_byte(widen_bits<T>(h[n])), at(n));
      return;
    }
  }
  uint32_t a[N];
#pragma unroll
  for (int n = 0; n < N; ++n) a[n] = abs_max_bits(v[n]);
  quantize_vecs<WHOLE>(v, a, at);
}

// A row is cut into units of 32 vectors.  Long rows: grid (rows, CTAs per row),
// a warp takes N units of a row, all in flight together.  (The bf16 form in
// vectors spills 12 bytes at its 64 registers, the bound that four CTAs set.)
constexpr int kQuantUnits = 4;

template <typename T, RowMode MODE>
__global__ void __launch_bounds__(256, MODE != ROW_ELEMENTS ? 4 : 1) quantize_rows_kernel(const RowsParams p) {
  constexpr int VEC = kRowVec<T>, N = kQuantUnits, STEP = 32 * VEC;
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t row = blockIdx.x;
  const int k = (int)p.k, chunk = (int)(blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5)) * N * STEP;
  if (chunk >= k) return;
  const int c = chunk + (int)(threadIdx.x & 31) * VEC;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  uint4 u[N];
#pragma unroll
  for (int n = 0; n < N; ++n) u[n] = load_vec<T, MODE>(x, c + n * STEP, k);
  uint8_t *q = p.q + row * p.q_ld + c, *s = p.s + row * p.s_ld + c / kFp8Block;
  auto at = [&](int n) { return VecPlace{q + n * STEP, s + n * (STEP / kFp8Block), k - c - n * STEP}; };
  if (chunk + N * STEP <= k) quantize_loaded<T, true>(u, at);
  else quantize_loaded<T, false>(u, at);
}

// Short rows, of `blocks` blocks: the lanes of a block take N blocks in turn,
// counted through all rows.
template <typename T, RowMode MODE>
__global__ void __launch_bounds__(256) quantize_short_kernel(const RowsParams p, const uint32_t blocks) {
  constexpr int VEC = kRowVec<T>, N = kQuantUnits, L = kFp8Block / VEC, B = 32 / L;  // L lanes per block
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * N * B, row0 = first / blocks;
  const int k = (int)p.k, lane = threadIdx.x & 31;
  const uint32_t b0 = (uint32_t)(first - row0 * blocks) + lane / L;
  auto place = [&](int n, int64_t& row, int& c) {
    const uint32_t b = b0 + n * B, r = b / blocks;
    row = row0 + r;
    c = row < p.m ? (int)((b - r * blocks) * kFp8Block + lane % L * VEC) : k;
  };
  uint4 u[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int64_t row;
    int c;
    place(n, row, c);
    u[n] = load_vec<T, MODE>(static_cast<const T*>(p.x) + row * p.x_ld, c, k);
  }
  quantize_loaded<T, false>(u, [&](int n) {
    int64_t row;
    int c;
    place(n, row, c);
    return VecPlace{p.q + row * p.q_ld + c, p.s + row * p.s_ld + c / kFp8Block, k - c};
  });
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

// Sum of squares in four partial sums.
struct SquareSum {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  template <int VEC>
  __device__ __forceinline__ void add(const float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      add_squares2(s[0], s[1], v[i], v[i + 1]);
      add_squares2(s[2], s[3], v[i + 2], v[i + 3]);
    }
  }
  __device__ __forceinline__ float total() const { return (s[0] + s[1]) + (s[2] + s[3]); }
};

template <int VEC>
__device__ __forceinline__ void add_vec(float (&v)[VEC], const float (&t)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i += 2) add2(v[i], v[i + 1], t[i], t[i + 1]);
}

// What follows once a row's h and scale are known: N vectors of it, vector n
// at column c + n step; k = 0 past the last row.
template <typename T, RowMode MODE, int N>
__device__ __forceinline__ void norm_finish(const RowsParams& p, int64_t row, int c, int step, int k, float scale,
                                            float (&v)[N][kRowVec<T>]) {
  constexpr int VEC = kRowVec<T>;
  if (p.h) {
#pragma unroll
    for (int n = 0; n < N; ++n) store_vec<T, MODE>(static_cast<T*>(p.h) + row * p.h_ld, c + n * step, k, v[n]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int at = c + n * step;
    if (!p.weight) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) mul2(v[n][i], v[n][i + 1], scale, scale);
    } else if (MODE == ROW_WHOLE || at < k) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 w = *reinterpret_cast<const float4*>(p.weight + at + i);
        mul2(v[n][i], v[n][i + 1], scale, scale);
        mul2(v[n][i + 2], v[n][i + 3], scale, scale);
        mul2(v[n][i], v[n][i + 1], w.x, w.y);
        mul2(v[n][i + 2], v[n][i + 3], w.z, w.w);
      }
    }
  }
  if (p.q) {
    uint32_t a[N];
#pragma unroll
    for (int n = 0; n < N; ++n) a[n] = abs_max_bits(v[n]);
    uint8_t *q = p.q + row * p.q_ld + c, *s = p.s + row * p.s_ld + c / kFp8Block;
    auto at = [&](int n) { return VecPlace{q + n * step, s + n * (step / kFp8Block), k - c - n * step}; };
    quantize_vecs<MODE == ROW_WHOLE>(v, a, at);
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) store_vec<T, MODE>(static_cast<T*>(p.y) + row * p.y_ld, c + n * step, k, v[n]);
  }
}

//   h = x + residual (fp32),  y = h / sqrt(mean(h^2) + eps) weight
// `lanes` threads per row, which keep it in registers: NV vectors per lane.  A
// row has 8 or 16 lanes of a warp (rows that short), or whole warps; a CTA has
// one row or several.  (The 16-bit forms of four vectors that may end past the
// row spill 20 bytes at their 64 registers, which 1024 threads allow.)
template <typename T, RowMode MODE, int NV>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const RowsParams p, const int lanes) {
  constexpr int VEC = kRowVec<T>;
  __shared__ float part[32];
  const int row_in_cta = (int)threadIdx.x / lanes, in_row = (int)threadIdx.x - row_in_cta * lanes;
  const int64_t row = (int64_t)blockIdx.x * ((int)blockDim.x / lanes) + row_in_cta;
  const int c0 = in_row * VEC, step = lanes * VEC, k = row < p.m ? (int)p.k : 0;
  grid_dep_wait();
  grid_dep_trigger();
  float v[NV][VEC];
  SquareSum sum;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = static_cast<const T*>(p.residual) + row * p.r_ld;
  uint4 xu[NV], ru[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) xu[j] = load_vec<T, MODE>(x, c0 + j * step, k);
  if (p.residual) {
#pragma unroll
    for (int j = 0; j < NV; ++j) ru[j] = load_vec<T, MODE>(r, c0 + j * step, k);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    unpack_vec<T>(xu[j], v[j]);
    if (p.residual) {
      float t[VEC];
      unpack_vec<T>(ru[j], t);
      add_vec(v[j], t);
    }
    sum.add(v[j]);
  }
  float ss = sum.total();
  for (int o = min(lanes, 32) / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lanes > 32) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = lanes >> 5;
    if (lane == 0) part[w] = ss;
    __syncthreads();
    ss = lane < warps ? part[row_in_cta * warps + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  const float scale = rsqrtf(ss / (float)p.k + p.eps);
  norm_finish<T, MODE>(p, row, c0, step, k, scale, v);
}

// One block of 128 columns held four elements per lane, 32 apart: its values
// by words, since a store of bytes costs what one of words does (16384 x 7001
// bf16 with a residual 285 us by bytes, 252 by words).  `c` is the lane's first
// column.  All of a warp call.
__device__ __forceinline__ void quantize_elements(float (&v)[4], uint8_t* q, uint8_t* s, int c, int k) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  a = __reduce_max_sync(0xffffffffu, a);
  if (a >= 0x7F800000u) {  // something not finite: the scale comes from the rest
    a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a = max(a, finite_abs_bits(v[i]));
      v[i] = nan_unless_finite(v[i]);
    }
    a = __reduce_max_sync(0xffffffffu, a);
  }
  const uint32_t byte = fp8_scale_byte(a), w = fp8_pack4(v[0], v[1], v[2], v[3], fp8_inv_scale(byte));
  // each lane four columns in a row: one from each of four lanes
  const int lane = threadIdx.x & 31, at = c + 3 * lane, from = 4 * (lane & 7), byte_at = lane >> 3;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __shfl_sync(0xffffffffu, w, from + i);
  const uint32_t two = byte_at | (byte_at + 4) << 4;
  const uint32_t word = __byte_perm(__byte_perm(b[0], b[1], two), __byte_perm(b[2], b[3], two), 0x5410);
  if (at + 4 <= k) {
    *reinterpret_cast<uint32_t*>(q + at) = word;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (at + i < k) q[at + i] = (uint8_t)(word >> (8 * i));
  }
  if (c % kFp8Block == 0 && c < k) s[c / kFp8Block] = (uint8_t)byte;
}

// h of NU blocks, held as above: c is the lane's first column.
template <typename T, int NU>
__device__ __forceinline__ void load_elements(const RowsParams& p, int64_t row, int c, int k, float (&v)[NU][4]) {
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld + c;
  const T* r = static_cast<const T*>(p.residual) + row * p.r_ld + c;
  T a[NU][4], b[NU][4];
  auto at = [](int n, int i) { return n * kFp8Block + 32 * i; };
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[n][i] = c + at(n, i) < k ? x[at(n, i)] : from_f32<T>(0.0f);
  if (p.residual) {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) b[n][i] = c + at(n, i) < k ? r[at(n, i)] : from_f32<T>(0.0f);
  }
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[n][i] = p.residual ? to_f32(a[n][i]) + to_f32(b[n][i]) : to_f32(a[n][i]);
}

// ... and its outputs.
template <typename T, int NU>
__device__ __forceinline__ void finish_elements(const RowsParams& p, int64_t row, int c, int k, float scale,
                                                float (&v)[NU][4]) {
  auto column = [&](int n, int i) { return c + n * kFp8Block + 32 * i; };
  auto store = [&](T* t) {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (column(n, i) < k) t[column(n, i)] = from_f32<T>(v[n][i]);
  };
  if (p.h) store(static_cast<T*>(p.h) + row * p.h_ld);
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[n][i] = v[n][i] * scale * (p.weight && column(n, i) < k ? p.weight[column(n, i)] : 1.0f);
  if (p.q) {
#pragma unroll
    for (int n = 0; n < NU; ++n) quantize_elements(v[n], p.q + row * p.q_ld, p.s + row * p.s_ld, column(n, 0), k);
  } else {
    store(static_cast<T*>(p.y) + row * p.y_ld);
  }
}

// The same where rows are not on 16-byte boundaries: element by element, lanes
// on consecutive elements, so that a warp's access is 64 or 128 bytes in a
// row.  A warp has NU quantisation blocks, four elements of each per lane, 32
// apart.  Bound by the number of accesses and by the loads in flight: 16384 x
// 7001 without residual 152 us in bf16 (46 % of the memory rate), 184 in fp32
// (76 %).  With eight or four consecutive elements per lane, a warp's accesses
// spread over four times the lines (373 and 302 us).  The quantise kernels
// above keep that order all the same: they store a lane's values as one word,
// and in this order take 122 us on that shape against 83 in bf16, 122 against
// 89 in fp32.
template <typename T, int NU>
__global__ void __launch_bounds__(1024) rms_norm_elements_kernel(const RowsParams p, const int warps) {
  __shared__ float part[32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int in_row = w % warps, first = w - in_row;
  const int64_t row = (int64_t)blockIdx.x * ((int)(blockDim.x >> 5) / warps) + w / warps;
  const int k = row < p.m ? (int)p.k : 0, c = in_row * NU * kFp8Block + lane;
  grid_dep_wait();
  grid_dep_trigger();
  float v[NU][4];
  load_elements<T>(p, row, c, k, v);
  SquareSum sum;
#pragma unroll
  for (int n = 0; n < NU; ++n) sum.add(v[n]);
  float ss = sum.total();
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (warps > 1) {
    if (lane == 0) part[w] = ss;
    __syncthreads();
    ss = lane < warps ? part[first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  finish_elements<T>(p, row, c, k, rsqrtf(ss / (float)p.k + p.eps), v);
}

// Rows too long for registers: one CTA per row, which reads it twice.
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const RowsParams p) {
  constexpr int VEC = kRowVec<T>, NU = 2;
  __shared__ float part[32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.r_ld : nullptr;
  const int64_t step = VECTORS ? 1024 * VEC : 32 * NU * kFp8Block;
  const int k = (int)p.k;
  using Values = float[VECTORS ? 1 : NU][VECTORS ? VEC : 4];  // a lane's part of a step
  auto load = [&](int c, Values& v) {
    if constexpr (VECTORS) {
      unpack_vec<T>(load_vec<T, ROW_VECTORS>(x, c, k), v[0]);
      if (r) {
        float t[VEC];
        unpack_vec<T>(load_vec<T, ROW_VECTORS>(r, c, k), t);
        add_vec(v[0], t);
      }
    } else {
      load_elements<T>(p, row, c, k, v);
    }
  };
  const int64_t c0 = w * (step / 32);  // a warp's first column; whole warps stay together to quantise
  const int in_warp = VECTORS ? lane * VEC : lane;
  SquareSum sum;
  for (int64_t c = c0; c < p.k; c += step) {
    Values v;
    load((int)c + in_warp, v);
#pragma unroll
    for (auto& u : v) sum.add(u);
  }
  float ss = sum.total();
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[w] = ss;
  __syncthreads();
  ss = part[lane];
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float scale = rsqrtf(ss / (float)p.k + p.eps);
  for (int64_t c = c0; c < p.k; c += step) {
    Values v;
    load((int)c + in_warp, v);
    if constexpr (VECTORS) norm_finish<T, ROW_VECTORS>(p, row, (int)c + in_warp, 0, k, scale, v);
    else finish_elements<T>(p, row, (int)c + in_warp, k, scale, v);
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
  const bool vec = p.k % kRowVec<T> == 0 && rows_vector<T>(p.x, p.x_ld, p.m);
  const int64_t units = (p.k + 32 * kRowVec<T> - 1) / (32 * kRowVec<T>);
  if (units < kQuantUnits) {
    const int64_t blocks = fp8_blocks(p.k), cta = 8 * kQuantUnits * 32 * kRowVec<T> / kFp8Block;
    return pdl_launch(vec ? quantize_short_kernel<T, ROW_VECTORS> : quantize_short_kernel<T, ROW_ELEMENTS>,
                      dim3((unsigned)((p.m * blocks + cta - 1) / cta)), dim3(256), 0, s, p, (uint32_t)blocks);
  }
  const int64_t warps = (units + kQuantUnits - 1) / kQuantUnits, ctas = (warps + 7) / 8;
  return pdl_launch(vec ? quantize_rows_kernel<T, ROW_VECTORS> : quantize_rows_kernel<T, ROW_ELEMENTS>,
                    dim3((unsigned)p.m, (unsigned)ctas), dim3((unsigned)(32 * ((warps + ctas - 1) / ctas))), 0, s, p);
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

template <typename T, RowMode MODE>
inline cudaError_t launch_rms_norm_m(const RowsParams& p, int nv, int lanes, cudaStream_t s) {
  const int rows = std::max(1, 256 / lanes);
  const unsigned grid = (unsigned)((p.m + rows - 1) / rows);
  return pdl_launch(nv == 4   ? rms_norm_kernel<T, MODE, 4>
                    : nv == 2 ? rms_norm_kernel<T, MODE, 2>
                              : rms_norm_kernel<T, MODE, 1>,
                    dim3(grid), dim3(rows * lanes), 0, s, p, lanes);
}
template <typename T>
inline cudaError_t launch_rms_norm_t(const RowsParams& p, int sm_count, cudaStream_t s) {
  const bool vec = p.k % kRowVec<T> == 0 && rows_vector<T>(p.x, p.x_ld, p.m) &&
                   rows_vector<T>(p.residual, p.r_ld, p.m) && rows_vector<T>(p.h, p.h_ld, p.m) &&
                   rows_vector<T>(p.y, p.y_ld, p.m) && (reinterpret_cast<uintptr_t>(p.weight) & 15) == 0;
  const int64_t vectors = (p.k + kRowVec<T> - 1) / kRowVec<T>;
  if (!vec) {
    const int64_t units = fp8_blocks(p.k);
    // Two passes above 128 blocks, which is what the registers of 1024 threads
    // hold, and in 16 bits, where the second pass finds more of the row in the
    // caches, above 64: 4096 x 12001 bf16 75 us in two passes, 92 in registers;
    // 16384 x 7001 bf16 191 and 152; 4096 x 16001 fp32 139 and 121.
    if (units > (sizeof(T) == 4 ? 128 : 64))
      return pdl_launch(rms_norm_long_kernel<T, false>, dim3((unsigned)p.m), dim3(1024), 0, s, p);
    // blocks per warp as the vectors below
    const int nu = units <= 32 && (p.m < 2 * sm_count || units == 1) ? 1 : units == 2 ? 2 : 4;
    const int warps = ((int)units + nu - 1) / nu, rows = std::max(1, 8 / warps);
    return pdl_launch(nu == 1   ? rms_norm_elements_kernel<T, 1>
                      : nu == 2 ? rms_norm_elements_kernel<T, 2>
                                : rms_norm_elements_kernel<T, 4>,
                      dim3((unsigned)((p.m + rows - 1) / rows)), dim3(32 * warps * rows), 0, s, p, warps);
  }
  if (vectors > 1024 * 4)  // more than the registers of 1024 threads hold
    return pdl_launch(rms_norm_long_kernel<T, true>, dim3((unsigned)p.m), dim3(1024), 0, s, p);
  // Many rows: up to four vectors per lane, so that few warps share a row and
  // many loads are in flight (16384 x 8192 bf16, residual, quantised: 149 us
  // with four, 200 with two, 241 with one).  Few rows: one per lane, the
  // shortest time (1 x 4096: 2.5 us against 3.4 with four).
  int nv = 1;
  if (p.m >= 2 * sm_count || vectors > 1024) nv = vectors <= 32 ? 1 : vectors <= 64 ? 2 : 4;
  // Whole warps, as many as the row needs (16384 x 5120 bf16, residual,
  // quantised: 87 us with five warps, 111 with eight), or the lanes of several
  // rows side by side in a warp.  A quantisation block's lanes stay together.
  const int need = (int)((vectors + nv - 1) / nv);
  int lanes = p.q ? kFp8Block / kRowVec<T> : 8;
  while (lanes < 32 && lanes < need) lanes *= 2;
  if (lanes < need) lanes = (need + 31) / 32 * 32;
  const int rows = std::max(1, 256 / lanes);
  if ((int64_t)lanes * nv == vectors && p.m % rows == 0) return launch_rms_norm_m<T, ROW_WHOLE>(p, nv, lanes, s);
  return launch_rms_norm_m<T, ROW_VECTORS>(p, nv, lanes, s);
}
inline cudaError_t launch_rms_norm(const RowsParams& p, int type, int sm_count, cudaStream_t s) {
  if (type == FTB_F32) return launch_rms_norm_t<float>(p, sm_count, s);
  if (type == FTB_F16) return launch_rms_norm_t<__half>(p, sm_count, s);
  return launch_rms_norm_t<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace ftb
