// Microscaled 4-bit floats (the OCP MX format with e2m1 values): blocks of 32 values along a row share a power-of-two
// scale.  Shared by the quantisation (mx4.hip) and the products (mx4_rows.hip, mx4_gemm.hip).
//
// Rows are kept as tiles of 16 rows by 128 values, each in the order a matrix instruction takes it: lane l of 64 has 32
// values (one block, 16 bytes, the value of the lower index in the low half of a byte) of row l % 16, the block l / 16 of the
// four.  A tile is 1024 bytes; tile (t, s) of rows 16t .. and values 128s .. is number t * steps + s, steps = K rounded up
// to 128, over 128.  So a tile is read as one piece wherever it goes.  The scales of four tiles one below the other (64
// rows) stand together, lane by lane, so that a lane's four are one dword: byte 256 * (t / 4 * steps + s) + 4 * l + t % 4.
// Rows and values past the last are zeros with scale byte 0, up to whole tiles and whole groups of four.
//
// A scale byte s stands for 2^(s - 127), 255 for NaN; s << 23 is the float32 that gfx950's conversions take for it, with 0
// read as 2^-127 and 255 giving NaN.
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
// Byte i of a dword of scales.
template <int I>
__device__ __forceinline__ float mx4_scale_of(uint32_t four) {
  return __uint_as_float((I == 3 ? four >> 1 : four << (23 - 8 * I)) & 0x7f800000u);
}
__device__ __forceinline__ float mx4_scale_of(uint32_t four, int i) {   // i known when unrolled
  return i == 0 ? mx4_scale_of<0>(four) : i == 1 ? mx4_scale_of<1>(four) : i == 2 ? mx4_scale_of<2>(four) : mx4_scale_of<3>(four);
}

__device__ __forceinline__ float mx4_gelu(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f)); }

}  // namespace ta
