// Products with 4-bit weights over many rows: Y[M, N] = epilogue(X[M, K] . W[N, K]^T) with X in bf16 (the weights made
// bf16, exactly, in front of the bf16 matrix instructions) or in 4 bits as well (v_mfma_scale_f32_16x16x128_f8f6f4 on the
// codes and scales as they are).  Sums are float32, the result is rounded once after the epilogue.
//
// A workgroup of four wavefronts computes a 128 x 128 tile, each wavefront 64 x 64 of it as 4 x 4 instruction tiles; K
// goes in steps of 128 through LDS, the next step's loads issued before a step is multiplied.  Rows and columns past the
// last repeat it and are not stored.
#include "mx4.hpp"

namespace ta {
namespace {

struct GemmArgs {
  const void* X;
  int64_t ldx;           // bf16: elements
  const uint32_t* XS;    // 4-bit X: its scales
  const uint4* W;
  const uint32_t* S;
  bf16_t* Y;
  int64_t ldy;
  const bf16_t* R;
  int64_t ldr;
  int M, N, K, Kp;
};

constexpr int BM = 128, BN = 128;

// 16-byte vector c of row r of a [rows][4] array of vectors: rotated within the row so that the 16 lanes that read one
// vector of 16 rows touch all banks
__device__ __forceinline__ int swz4(int r, int c) { return r * 4 + (c ^ ((r >> 2) & 3)); }
// the same for [rows][16]
__device__ __forceinline__ int swz16(int r, int c) { return r * 16 + (c ^ (r & 15)); }

template <bool BOTH, int EPI>
__global__ __launch_bounds__(256) void mx4_gemm_kernel(GemmArgs a) {
  constexpr int XV = BOTH ? 4 : 16;              // 16-byte vectors of a row of X in a step
  __shared__ uint4 xs[BM * XV];
  __shared__ uint4 ws[BN * 4];
  const int tid = threadIdx.x, lane = lane_id(), w = wave_id();
  const int li = lane & 15, lg = lane >> 4;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const int wm = (w & 1) * 64, wn = (w >> 1) * 64;
  const int ks = a.Kp / 128;

  uint4 xr[XV / 2], wr[2];                       // 256 threads: BM * XV / 256 and BN * 4 / 256 vectors each
  auto load = [&](int st) {
#pragma unroll
    for (int j = 0; j < XV / 2; ++j) {
      const int i = j * 256 + tid, r = i / XV, c = i % XV;
      const int m = m0 + r < a.M ? m0 + r : a.M - 1;
      if constexpr (BOTH) {
        xr[j] = ldg16(reinterpret_cast<const uint4*>(a.X) + (int64_t)m * ks * 4 + st * 4 + c);
      } else {
        const int k = st * 128 + c * 8;
        xr[j] = make_uint4(0, 0, 0, 0);
        if (k < a.K) xr[j] = ldg16(reinterpret_cast<const bf16_t*>(a.X) + (int64_t)m * a.ldx + k);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = j * 256 + tid, r = i / 4, c = i % 4;
      const int n = n0 + r < a.N ? n0 + r : a.N - 1;
      wr[j] = ldg16(a.W + (int64_t)n * ks * 4 + st * 4 + c);
    }
  };
  uint32_t sw[4], sx[4];
  const uint32_t *pw[4], *px[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = n0 + wn + c * 16 + li, m = m0 + wm + c * 16 + li;
    pw[c] = a.S + (int64_t)(n < a.N ? n : a.N - 1) * ks;
    if constexpr (BOTH) px[c] = a.XS + (int64_t)(m < a.M ? m : a.M - 1) * ks;
  }

  f32x4_t acc[4][4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  load(0);
  for (int st = 0; st < ks; ++st) {
    if (st > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < XV / 2; ++j) {
      const int i = j * 256 + tid, r = i / XV, c = i % XV;
      xs[BOTH ? swz4(r, c) : swz16(r, c)] = xr[j];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = j * 256 + tid;
      ws[swz4(i / 4, i % 4)] = wr[j];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      sw[c] = pw[c][st];
      if constexpr (BOTH) sx[c] = px[c][st];
    }
    __syncthreads();
    if (st + 1 < ks) load(st + 1);
    uint4 wq[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) wq[c] = ws[swz4(wn + c * 16 + li, lg)];
    if constexpr (BOTH) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint4 xq = xs[swz4(wm + m * 16 + li, lg)];
        const i32x8_t av = {(int)xq.x, (int)xq.y, (int)xq.z, (int)xq.w, 0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const i32x8_t bv = {(int)wq[c].x, (int)wq[c].y, (int)wq[c].z, (int)wq[c].w, 0, 0, 0, 0};
          acc[m][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[m][c], 4, 4, 0, sx[m] >> (8 * lg),
                                                                       0, sw[c] >> (8 * lg));
        }
      }
    } else {
      float sc[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[c] = mx4_scale((sw[c] >> (8 * lg)) & 255u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bf16x8_t bw[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          bw[c] = mx4_bf16x8(u == 0 ? wq[c].x : u == 1 ? wq[c].y : u == 2 ? wq[c].z : wq[c].w, sc[c]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint4 xq = xs[swz16(wm + m * 16 + li, lg * 4 + u)];
          const bf16x8_t ax = __builtin_bit_cast(bf16x8_t, xq);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ax, bw[c], acc[m][c], 0, 0, 0);
        }
      }
    }
  }

#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + wm + m * 16 + lg * 4 + i;
      if (row >= a.M) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = n0 + wn + c * 16 + li;
        if (n >= a.N) continue;
        float s = acc[m][c][i];
        if constexpr (EPI == MX_EPI_GELU) s = mx4_gelu(s);
        if constexpr (EPI == MX_EPI_RESIDUAL) s += to_f32(a.R[(int64_t)row * a.ldr + n]);
        a.Y[(int64_t)row * a.ldy + n] = bf16_from(s);
      }
    }
}

template <bool BOTH>
int launch_gemm(const GemmArgs& a, int epilogue, hipStream_t st) {
  const dim3 grid((a.N + BN - 1) / BN, (a.M + BM - 1) / BM), blk(256);
  if (grid.y > 65535) {
    set_error("mx4 product: too many rows (at most 8388480)");
    return TA_ERR_UNSUPPORTED;
  }
  switch (epilogue) {
    case MX_EPI_NONE: hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MX_EPI_NONE>), grid, blk, 0, st, a); break;
    case MX_EPI_GELU: hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MX_EPI_GELU>), grid, blk, 0, st, a); break;
    default: hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MX_EPI_RESIDUAL>), grid, blk, 0, st, a); break;
  }
  return check_launch("mx4_gemm_kernel");
}

}  // namespace

int mx4_gemm_bf16(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy, const void* R,
                  int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st) {
  GemmArgs a{X, ldx, nullptr, (const uint4*)Wp, (const uint32_t*)Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr, M, N, K,
             mx4_padded(K)};
  return launch_gemm<false>(a, epilogue, st);
}

}  // namespace ta

using namespace ta;

extern "C" int ta_mx4_both(const void* Xp, const uint8_t* Xs, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                           const void* R, int64_t ldr, int M, int N, int K, int epilogue, void* stream) {
  if (M < 0 || N < 1 || K < 1 || K > 0x7fffff00 || (M > 1 && ldy < N) || epilogue < 0 || epilogue > 2 ||
      (epilogue == MX_EPI_RESIDUAL && (R == nullptr || (M > 1 && ldr < N)))) {
    set_error("ta_mx4_both: bad sizes (a residual needs its rows)");
    return TA_ERR_ARG;
  }
  if (M == 0) return TA_OK;
  if (Xp == nullptr || Xs == nullptr || Wp == nullptr || Ws == nullptr || Y == nullptr ||
      ((uintptr_t)Xp | (uintptr_t)Wp) % 16 || ((uintptr_t)Xs | (uintptr_t)Ws) % 4 || (uintptr_t)Y % 2) {
    set_error("ta_mx4_both: packed rows must be 16-byte aligned, scales 4-byte aligned");
    return TA_ERR_ARG;
  }
  GemmArgs a{Xp, 0, (const uint32_t*)Xs, (const uint4*)Wp, (const uint32_t*)Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr,
             M, N, K, mx4_padded(K)};
  return launch_gemm<true>(a, epilogue, (hipStream_t)stream);
}
