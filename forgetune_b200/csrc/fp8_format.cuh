// The block-scaled 8-bit format and the types at its edges.
//
// A quantised row holds e4m3 values q and, for each block of 128 along the
// row, one scale s = 2^e stored as the byte e + 127 (ue8m0, the format the
// tensor cores take scales in); the block stands for q s.  Weights share one
// scale per 128 x 128 block.  The scale is the smallest power of two with
// max|x| / s <= 448, the largest e4m3 value, so a value is rounded once, to
// nearest even, and never saturates: x / s is exact (s is a power of two).
// A power of two costs no accuracy against max|x| / 448 as the scale, because
// e4m3 rounds relative to the value itself, except for values below 2^-6 s.
// A block of zeros has the scale 1.  Values that are not finite become NaN;
// the scale comes from the finite ones.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "forgetune_b200.h"

namespace ftb {

constexpr int kFp8Block = 128;
constexpr int kFp8Type = 3;  // beside FTB_F32 .. FTB_BF16: a quantised output

inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// |v| as ordered bits, 0 where v is not finite.
__device__ __forceinline__ uint32_t finite_abs_bits(float v) {
  const uint32_t a = __float_as_uint(v) & 0x7FFFFFFFu;
  return a < 0x7F800000u ? a : 0u;
}

// The scale byte of a block whose largest |x| has these bits.  448 is
// 1.75 2^8: with |x| = 1.f 2^p the exponent is p - 8, one more when
// 1.f > 1.75.  Below 2^-119 it stays at the smallest, 2^-127.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits) {
  if (amax_bits == 0u) return 127u;
  const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)(b > 0 ? b : 0);
}

// 1 / scale = 2^(127 - byte), exact: the byte is at most 247.
__device__ __forceinline__ float fp8_inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Keeps every finite v (signed zeros too) and turns infinities into NaN,
// which the saturating conversion would make 448.
__device__ __forceinline__ float nan_unless_finite(float v) { return __fmaf_rn(v, 0.0f, v); }

// Two fp32 operations in one instruction, each rounded as usual.  The kernels
// over rows are short of issue slots when the power limit lowers the clock.
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\t"
      "mul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\t"
      "add.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
// (s, t) += (a a, b b)
__device__ __forceinline__ void add_squares2(float& s, float& t, float a, float b) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\t"
      "fma.rn.f32x2 p, q, q, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(s), "+f"(t)
      : "f"(a), "f"(b));
}

// Four values (finite or NaN) over the scale as e4m3, the first in the lowest byte.
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inv) {
  mul2(a, b, inv, inv);
  mul2(c, d, inv, inv);
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

}  // namespace ftb
