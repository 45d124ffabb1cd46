// Rounding rows to microscaled 4-bit floats (mx4.hpp).
//
// A block of 32 values with largest magnitude a takes the scale 2^e, e = floor(log2 a) - 2 (the exponent of e2m1's
// largest number, 6, being 2), so the scaled values lie in (-8, 8); each is rounded to the nearest of 0, .5, 1, 1.5, 2,
// 3, 4, 6 (ties to the even code) and saturates at 6.  Scaling by a power of two is exact.
//
// Bound by the bytes: 16384 x 4096 float32 with its rounded values written beside the codes (573 MB) in 118 us, 4.9 TB/s
// (a large copy reaches 5.1 to 5.7 here); 37 x 1000 bf16 3.3 us, a launch and a round trip.  Eight values a thread are one
// or two 16-byte loads and one dword of codes, a block's largest magnitude two exchanges between neighbouring lanes.
#include "mx4.hpp"

namespace ta {
namespace {

// A workgroup takes a tile after another: thread i eight values (i % 16) of row i / 16, four threads a block.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx4_quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int steps,
                                                        int64_t tiles, uint32_t* __restrict__ packed,
                                                        uint8_t* __restrict__ scale, T* __restrict__ values, int64_t ldv) {
  const int li = threadIdx.x / 16, j = threadIdx.x % 16;
  const int64_t last = (rows - 1) / 16;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t rt = steps == 1 ? t : t / steps;
    const int64_t row = rt * 16 + li;
    const int c0 = (int)(t - rt * steps) * 128 + j * 8;
    const bool in = row < rows;
    const T* xr = x + (in ? row : 0) * ldx + c0;
    float f[8];
    if (VEC && in && c0 + 8 <= K) {
      load_row_g<T, 8>(xr, f);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] = in && c0 + u < K ? to_f32(xr[u]) : 0.0f;
    }
    float a = 0.0f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      a = fmaxf(a, fabsf(f[u]));
      bad |= !(fabsf(f[u]) < INFINITY);
    }
    a = bad ? INFINITY : a;
    a = fmaxf(a, dpp_f<0xB1>(a));   // the four threads of the block
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
    const int l = (j / 4) * 16 + li;   // the lane whose block this is
    packed[t * 256 + l * 4 + j % 4] = w;
    if (j % 4 == 0) {
      uint8_t* sc = scale + ((rt >> 2) * steps + (t - rt * steps)) * 256 + l * 4;
      sc[rt & 3] = (uint8_t)byte;
      if (rt == last)
        for (int i = (int)(rt & 3) + 1; i < 4; ++i) sc[i] = 0;   // the rest of the last group
    }
    if (values != nullptr && in) {
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
  const int steps = mx4_padded(K) / 128;
  const int64_t tiles = (rows + 15) / 16 * steps;
  const unsigned grid = (unsigned)(tiles < (1 << 20) ? tiles : (1 << 20));
  const int sz = (int)sizeof(T);
  const bool vec = (uintptr_t)x % 16 == 0 && (ldx * sz) % 16 == 0 &&
                   (values == nullptr || ((uintptr_t)values % 16 == 0 && (ldv * sz) % 16 == 0));
  if (vec)
    hipLaunchKernelGGL((mx4_quant_kernel<T, true>), dim3(grid), dim3(256), 0, st, (const T*)x, ldx, rows, K, steps, tiles,
                       (uint32_t*)packed, scale, (T*)values, ldv);
  else
    hipLaunchKernelGGL((mx4_quant_kernel<T, false>), dim3(grid), dim3(256), 0, st, (const T*)x, ldx, rows, K, steps, tiles,
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
