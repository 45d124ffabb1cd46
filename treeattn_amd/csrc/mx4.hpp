// Microscaled 4-bit floats (the OCP MX format with e2m1 values): blocks of 32 values along a row share a power-of-two
// scale.  Shared by the quantisation (mx4.hip) and the products (mx4_rows.hip, mx4_gemm.hip).
//
// A row of K values is Kp = K rounded up to 128 values long: Kp / 2 bytes, the value of the lower index in the low half
// of a byte, and Kp / 32 scale bytes, so a block is one 16-byte vector and four blocks one dword of scales.  A scale byte
// s stands for 2^(s - 127), 255 for NaN; s << 23 is the float32 that gfx950's conversions take for it, with 0 read as
// 2^-127 and 255 giving NaN.
#pragma once

#include "common.hpp"

namespace ta {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

enum { MX_EPI_NONE = 0, MX_EPI_GELU = 1, MX_EPI_RESIDUAL = 2 };

__host__ __device__ __forceinline__ int mx4_padded(int K) { return (K + 127) & ~127; }

// Eight values (one dword of codes) as bf16, exactly: |value| <= 6 times a power of two.
__device__ __forceinline__ bf16x8_t mx4_bf16x8(uint32_t codes, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ float mx4_gelu(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f)); }

}  // namespace ta
