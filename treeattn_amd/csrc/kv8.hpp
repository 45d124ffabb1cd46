// A decode cache in 8 bits: pages of one leaf block of one (sequence, head), each with a scale for its keys and one
// for its values, and the block being filled kept unrounded beside them.  Shared by the kernels that write it
// (kv8.hip) and the attention that reads it (attend8.hip).
#pragma once

#include "common.hpp"

namespace ta {

// Device view of a ta_kv8 (include/treeattn.h).  Page p: K rows at pool + p * 2 * leaf * D, V rows leaf * D bytes
// further; scale[2p] of the keys, scale[2p + 1] of the values.  The unrounded block of (b, h): K rows at
// tail + b * tail_sb + h * tail_sh, V rows leaf * D elements further; tail_block[b * tb_sb + h] says which leaf block
// it is (-1: none).
struct Kv8 {
  uint8_t* pool;
  float* scale;
  const int32_t* table;
  int64_t sb, sh;
  int64_t npages;
  void* tail;
  int64_t tail_sb, tail_sh;
  int32_t* tail_block;
  int64_t tb_sb;
  int blog2;
  int tcap;
  // the page of leaf block j of the (sequence, head) whose table row this is, -1 when it has none
  __device__ __forceinline__ int page(const int32_t* row, int j) const {
    const int pg = row[j];
    return pg >= 0 && pg < npages ? pg : -1;
  }
};

// Checks a description against the head size and the dtype of its unrounded block (TA_OK, or an error that names
// `who`).
int kv8_view(const ta_kv8* c, int dtype, int B, int H, int D, const char* who, Kv8& out);

// 16 bytes of e4m3 -> 16 floats
__device__ __forceinline__ void e4m3_x16(const uint4& u, float (&f)[16]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    f[4 * i] = a.x;
    f[4 * i + 1] = a.y;
    f[4 * i + 2] = b.x;
    f[4 * i + 3] = b.y;
  }
}

// A page's value (an e4m3 number times its scale), or a mean of such values, in the model's type.  A magnitude near float16's
// largest, 65504, is rounded up to 65536 in a page; what passes the range that way is the largest number, not infinity.
template <typename T>
__device__ __forceinline__ T page_value(float x) {
  if constexpr (__is_same(T, f16_t)) x = fabsf(x) > 65504.0f && fabsf(x) < INFINITY ? copysignf(65504.0f, x) : x;
  return from_f32<T>(x);
}

// A finite magnitude, 0 for what is not finite: what a scale is chosen from.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

// The exponent of the scale of values whose largest finite magnitude is amax: the smallest e in [-126, 127] with
// amax <= 448 * 2^e (448 = 0.875 * 2^9 is the largest e4m3 number), 0 for amax = 0.
__device__ __forceinline__ int e4m3_exponent(float amax) {
  if (!(amax > 0.0f)) return 0;
  int x;
  const float m = frexpf(amax, &x);   // amax = m * 2^x, m in [0.5, 1)
  const int e = x - 9 + (m > 0.875f ? 1 : 0);
  return e < -126 ? -126 : (e > 127 ? 127 : e);
}

// Four values times 2^-e as e4m3, rounded to nearest even; what is not finite becomes NaN.  The product is exact (a
// power of two, |result| <= 448; only results below 2^-126 lose bits, and those round to zero).
__device__ __forceinline__ uint32_t e4m3_x4(float a, float b, float c, float d, int e) {
  const float v[4] = {a, b, c, d};
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = fabsf(v[i]) < INFINITY ? ldexpf(v[i], -e) : __builtin_nanf("");
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
}

}  // namespace ta
