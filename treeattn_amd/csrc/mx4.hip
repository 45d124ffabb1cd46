// Rounding rows to microscaled 4-bit floats (mx4.hpp).
//
// A block of 32 values with largest magnitude a takes the scale 2^e, e = floor(log2 a) - 2 (the exponent of e2m1's
// largest number, 6, being 2), so the scaled values lie in (-8, 8); each is rounded to the nearest of 0, .5, 1, 1.5, 2,
// 3, 4, 6 (ties to the even code) and saturates at 6.  Scaling by a power of two is exact.
#include "mx4.hpp"

namespace ta {
namespace {

// Eight consecutive values of a row per lane, four lanes per block.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx4_quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K,
                                                        uint32_t* __restrict__ packed, uint8_t* __restrict__ scale,
                                                        T* __restrict__ values, int64_t ldv) {
  const int per = mx4_padded(K) / 8;   // groups of eight in a row
  const int64_t total = rows * per;
  const int64_t step = (int64_t)gridDim.x * 256;
  // (total is a multiple of 16, so the four lanes of a block leave the loop together)
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += step) {
    const int64_t row = i / per;
    const int c0 = (int)(i - row * per) * 8;
    const T* xr = x + row * ldx + c0;
    float f[8];
    if (VEC && c0 + 8 <= K) {
      load_row_g<T, 8>(xr, f);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = c0 + u < K ? to_f32(xr[u]) : 0.0f;
    }
    float a = 0.0f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      a = fmaxf(a, fabsf(f[u]));
      bad |= !(fabsf(f[u]) < INFINITY);
    }
    a = bad ? INFINITY : a;
    a = fmaxf(a, dpp_f<0xB1>(a));   // the four lanes of the block
    a = fmaxf(a, dpp_f<0x4E>(a));
    bad = !(a < INFINITY);
    int e = -127;
    if (a > 0.0f && !bad) {
      int ex;
      (void)frexpf(a, &ex);   // floor(log2 a) = ex - 1
      e = ex - 3 > -127 ? ex - 3 : -127;
    }
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);   // 2^-e: e is in [-127, 125]
    uint32_t w = 0;
    if (!bad) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * inv, f[1] * inv, 1.0f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * inv, f[3] * inv, 1.0f, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4] * inv, f[5] * inv, 1.0f, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6] * inv, f[7] * inv, 1.0f, 3);
    }
    const uint32_t byte = bad ? 255u : (uint32_t)(e + 127);
    packed[i] = w;
    if ((i & 3) == 0) scale[i >> 2] = (uint8_t)byte;
    if (values != nullptr) {
      const float s = mx4_scale(byte);
      f32x2_t v[4];
      v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
      v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
      v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
      v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
      T o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) o[u] = from_f32<T>(u & 1 ? v[u / 2].y : v[u / 2].x);
      T* vr = values + row * ldv + c0;
      if (VEC && c0 + 8 <= K) {
#pragma unroll
        for (int u = 0; u < 8; u += 16 / (int)sizeof(T))
          *reinterpret_cast<uint4*>(vr + u) = *reinterpret_cast<const uint4*>(o + u);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (c0 + u < K) vr[u] = o[u];
      }
    }
  }
}

template <typename T>
int launch_quant(const void* x, int64_t ldx, int64_t rows, int K, void* packed, uint8_t* scale, void* values,
                 int64_t ldv, hipStream_t st) {
  const int64_t groups = rows * (mx4_padded(K) / 8);
  const int64_t want = (groups + 255) / 256;
  const unsigned grid = (unsigned)(want < (1 << 20) ? want : (1 << 20));
  const int sz = (int)sizeof(T);
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * sz) % 16 == 0 &&
                   (values == nullptr || ((uintptr_t)values % 16 == 0 && (ldv * sz) % 16 == 0));
  if (vec)
    hipLaunchKernelGGL((mx4_quant_kernel<T, true>), dim3(grid), dim3(256), 0, st, (const T*)x, ldx, rows, K,
                       (uint32_t*)packed, scale, (T*)values, ldv);
  else
    hipLaunchKernelGGL((mx4_quant_kernel<T, false>), dim3(grid), dim3(256), 0, st, (const T*)x, ldx, rows, K,
                       (uint32_t*)packed, scale, (T*)values, ldv);
  return check_launch("mx4_quant_kernel");
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_mx4_quant(const void* x, int dtype, int64_t ldx, int64_t rows, int K, void* packed, uint8_t* scale,
                            void* values, int64_t ldv, void* stream) {
  if (rows < 0 || K < 1 || K > 0x7fffff00 || (rows > 1 && ldx < 0) || (rows > 0 && (x == nullptr || packed == nullptr || scale == nullptr)) ||
      (uintptr_t)packed % 16 || (uintptr_t)scale % 4 || (values != nullptr && rows > 1 && ldv < K)) {
    set_error("ta_mx4_quant: bad sizes (K at least 1), a missing pointer, or packed / scale not 16- / 4-byte aligned");
    return TA_ERR_ARG;
  }
  if (rows == 0) return TA_OK;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case TA_F32: return launch_quant<float>(x, ldx, rows, K, packed, scale, values, ldv, st);
    case TA_F16: return launch_quant<f16_t>(x, ldx, rows, K, packed, scale, values, ldv, st);
    case TA_BF16: return launch_quant<bf16_t>(x, ldx, rows, K, packed, scale, values, ldv, st);
    default: set_error("ta_mx4_quant: unknown dtype"); return TA_ERR_ARG;
  }
}
