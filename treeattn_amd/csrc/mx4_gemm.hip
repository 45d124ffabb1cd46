// Products with 4-bit weights over many rows: Y[M, N] = epilogue(X[M, K] . W[N, K]^T) with X in bf16 (the weights made
// bf16, exactly, in front of the bf16 matrix instructions) or in 4 bits as well (v_mfma_scale_f32_16x16x128_f8f6f4 on the
// codes and scales as they are).  Sums are float32, the result is rounded once after the epilogue.
//
// A workgroup of eight wavefronts, two along M by four along N, computes a (32 MT) x (64 NT) tile; a wavefront MT x NT
// instruction tiles of it.  K goes through LDS in steps of 256 (both in 4 bits) or 64 (bf16 X): 128 bytes a row of X,
// copied straight from memory to LDS, the next step's copies in flight while a step is multiplied.  The weights are the
// instructions' first operand, so a lane ends with four consecutive columns of one row.
//
// k inside a step is dealt so that a lane's operands lie together: with both in 4 bits, lane group g = lane / 16 takes
// blocks 2g and 2g + 1 of the step's eight, so two scale bytes that lie together serve its two instructions; with bf16 X
// it takes k = 16g .. 16g + 15, half a block (eight bytes of codes, one scale).  X and W agree, so any order is right.
// Rows and columns past the last repeat it and are not stored; what a step has past K is read as zeros.
#include "mx4.hpp"

namespace ta {
namespace {

struct GemmArgs {
  const char* X;         // rows of xb bytes
  int64_t xb;
  const uint32_t* XS;    // 4-bit X: its scales, Kp / 128 dwords a row
  const char* W;         // rows of Kp / 2 bytes
  const uint32_t* S;
  bf16_t* Y;
  int64_t ldy;
  const bf16_t* R;
  int64_t ldr;
  int M, N, K, Kp;
  int tm, tn;            // tiles along M and N
  int vec;               // Y and R take 8-byte accesses
};

constexpr int kGemmThreads = 512;
// What copies past the end of a row read.
__device__ const uint4 kZeros = {0, 0, 0, 0};

// Slot of 16-byte vector c of row r in an LDS array of rows of eight: rotated so that the 16 lanes that read one vector
// of 16 consecutive rows touch all banks.
__device__ __forceinline__ int slot8(int r, int c) { return r * 8 + (c ^ ((r >> 1) & 7)); }
// The same for rows of two vectors read in halves.
__device__ __forceinline__ int slot2(int r, int c) { return r * 2 + (c ^ ((r >> 3) & 1)); }

__device__ __forceinline__ void to_lds16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)dst, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)dst, 4, 0, 0);
}

template <bool BOTH, int MT, int NT>
struct GemmTile {
  static constexpr int BM = 32 * MT, BN = 64 * NT;
  static constexpr int STEP = BOTH ? 256 : 64;                // of K
  static constexpr int XB = BM * 128;                         // LDS bytes of X a step
  static constexpr int WB = BOTH ? BN * 128 : BN * 32;        // of W
  static constexpr int SB = BOTH ? (BM + BN) * 8 : BN * 4;    // of scales (bf16 X: of two steps)
  static constexpr int LDS = 2 * (XB + WB + SB);
};

template <bool BOTH, int MT, int NT, int EPI>
__global__ __launch_bounds__(kGemmThreads) void mx4_gemm_kernel(GemmArgs a) {
  using G = GemmTile<BOTH, MT, NT>;
  constexpr int BM = G::BM, BN = G::BN;
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), w = wave_id();
  const int li = lane & 15, lg = lane >> 4;
  const int wm = (w & 1) * 16 * MT, wn = (w >> 1) * 16 * NT;
  // Workgroups go to the eight XCDs in turn: each XCD takes a contiguous run of tiles, in groups of eight rows of tiles,
  // so that what its workgroups share stays in its L2.
  int m0, n0;
  {
    const int T = a.tm * a.tn, id = blockIdx.x, x = id & 7, q = T >> 3, r = T & 7;
    const int t = x * q + (x < r ? x : r) + (id >> 3);
    const int per = 8 * a.tn, g = t / per, gm = a.tm - g * 8 < 8 ? a.tm - g * 8 : 8;
    m0 = (g * 8 + (t - g * per) % gm) * BM;
    n0 = (t - g * per) / gm * BN;
  }
  const int kd = a.Kp / 128;                                  // scale dwords of a row
  const int steps = BOTH ? (a.Kp + 255) / 256 : (a.K + 63) / 64;

  // byte offsets, from the tile's first row, of what this lane copies
  const char* xbase = a.X + (int64_t)m0 * a.xb;
  const char* wbase = a.W + (int64_t)n0 * (a.Kp / 2);
  constexpr int NX = BM * 8 / kGemmThreads;                   // copies of X a wavefront and step
  constexpr int NW = BOTH ? BN * 8 / kGemmThreads : 1;
  constexpr int NS = BOTH ? (BM + BN) * 2 / kGemmThreads : 1;
  uint32_t xo[NX], wo[NW];
  int xc[NX], wc[NW];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int s = (i * 8 + w) * 64 + lane, r = s / 8;
    xc[i] = (s % 8) ^ ((r >> 1) & 7);
    xo[i] = (uint32_t)(m0 + r < a.M ? r : a.M - 1 - m0) * (uint32_t)a.xb + xc[i] * 16;
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int s = (i * 8 + w) * 64 + lane;
    const int r = BOTH ? s / 8 : s / 2;
    wc[i] = BOTH ? (s % 8) ^ ((r >> 1) & 7) : (s % 2) ^ ((r >> 3) & 1);
    wo[i] = (uint32_t)(n0 + r < a.N ? r : a.N - 1 - n0) * (uint32_t)(a.Kp / 2) + wc[i] * 16;
  }
  const uint32_t* sp[NS];
  int sd[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int s = (i * 8 + w) * 64 + lane;
    if constexpr (BOTH) {
      const int r = s / 2;
      sd[i] = s & 1;
      sp[i] = r < BM ? a.XS + (int64_t)(m0 + r < a.M ? m0 + r : a.M - 1) * kd + sd[i]
                     : a.S + (int64_t)(n0 + r - BM < a.N ? n0 + r - BM : a.N - 1) * kd + sd[i];
    } else {
      sd[i] = 0;
      sp[i] = a.S + (int64_t)(n0 + s < a.N ? n0 + s : a.N - 1) * kd;
    }
  }
  const bool ragged = BOTH ? (a.Kp & 255) != 0 : (a.K & 63) != 0;

  auto lx = [&](int buf) { return lds + buf * G::XB; };
  auto lw = [&](int buf) { return lds + 2 * G::XB + buf * G::WB; };
  auto ls = [&](int buf) { return lds + 2 * (G::XB + G::WB) + buf * G::SB; };

  auto stage = [&](int s, int buf) {
    const bool last = ragged && s == steps - 1;
    const char* xs = xbase + (int64_t)s * 128;
    const char* ws = wbase + (int64_t)s * (BOTH ? 128 : 32);
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const void* src = xs + xo[i];
      if (last && (BOTH ? s * 8 + xc[i] >= kd * 4 : s * 64 + xc[i] * 8 >= a.K)) src = &kZeros;
      to_lds16(src, lx(buf) + (i * 8 + w) * 1024);
    }
    if constexpr (BOTH) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const void* src = ws + wo[i];
        if (last && s * 8 + wc[i] >= kd * 4) src = &kZeros;
        to_lds16(src, lw(buf) + (i * 8 + w) * 1024);
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const void* src = sp[i] + s * 2;
        if (last && s * 2 + sd[i] >= kd) src = &kZeros;
        to_lds4(src, ls(buf) + (i * 8 + w) * 256);
      }
    } else {
      if (w < BN / 32) to_lds16(ws + wo[0], lw(buf) + w * 1024);
      if ((s & 1) == 0 && w < BN / 64) to_lds4(sp[0] + (s >> 1), ls((s >> 1) & 1) + w * 256);
    }
  };

  f32x4_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto multiply = [&](int s, int buf) {
    const uint4* x = reinterpret_cast<const uint4*>(lx(buf));
    if constexpr (BOTH) {
      const uint4* wl = reinterpret_cast<const uint4*>(lw(buf));
      const uint16_t* sc = reinterpret_cast<const uint16_t*>(ls(buf));
      uint4 wq[NT][2];
      int sw[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int r = wn + c * 16 + li;
        sw[c] = sc[(BM + r) * 4 + lg];
#pragma unroll
        for (int k = 0; k < 2; ++k) wq[c][k] = wl[slot8(r, lg * 2 + k)];
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = wm + m * 16 + li;
        const int sx = sc[r * 4 + lg];
        uint4 xq[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) xq[k] = x[slot8(r, lg * 2 + k)];
        const i32x8_t x0 = {(int)xq[0].x, (int)xq[0].y, (int)xq[0].z, (int)xq[0].w, 0, 0, 0, 0};
        const i32x8_t x1 = {(int)xq[1].x, (int)xq[1].y, (int)xq[1].z, (int)xq[1].w, 0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const i32x8_t w0 = {(int)wq[c][0].x, (int)wq[c][0].y, (int)wq[c][0].z, (int)wq[c][0].w, 0, 0, 0, 0};
          acc[m][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w0, x0, acc[m][c], 4, 4, 0, sw[c], 0, sx);
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const i32x8_t w1 = {(int)wq[c][1].x, (int)wq[c][1].y, (int)wq[c][1].z, (int)wq[c][1].w, 0, 0, 0, 0};
          acc[m][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w1, x1, acc[m][c], 4, 4, 1, sw[c], 1, sx);
        }
      }
    } else {
      const uint2* wl = reinterpret_cast<const uint2*>(lw(buf));
      const uint8_t* sc = reinterpret_cast<const uint8_t*>(ls((s >> 1) & 1)) + 2 * (s & 1) + (lg >> 1);
      bf16x8_t wv[NT][2];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int r = wn + c * 16 + li;
        const uint2 q = wl[slot2(r, lg >> 1) * 2 + (lg & 1)];
        const float f = mx4_scale(sc[r * 4]);
        wv[c][0] = mx4_bf16x8(q.x, f);
        wv[c][1] = mx4_bf16x8(q.y, f);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = wm + m * 16 + li;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const bf16x8_t xv = __builtin_bit_cast(bf16x8_t, x[slot8(r, lg * 2 + k)]);
#pragma unroll
          for (int c = 0; c < NT; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[c][k], xv, acc[m][c], 0, 0, 0);
        }
      }
    }
  };

  stage(0, 0);
  for (int s = 0; s < steps; ++s) {
    wait_vmcnt_n<0>();   // this wavefront's copies of step s have landed
    __syncthreads();     // everyone's have, and everyone is done with the buffer the next copies fill
    if (s + 1 < steps) stage(s + 1, (s + 1) & 1);
    multiply(s, s & 1);
  }

  // element (row n, col m) of an instruction tile is register n % 4 of lane (n / 4) * 16 + m
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = m0 + wm + m * 16 + li;
    if (row >= a.M) continue;
    bf16_t* yr = a.Y + (int64_t)row * a.ldy;
    const bf16_t* rr = a.R + (int64_t)row * a.ldr;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const int n = n0 + wn + c * 16 + lg * 4;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = acc[m][c][i];
      if constexpr (EPI == MX_EPI_GELU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = mx4_gelu(f[i]);
      }
      if (a.vec && n + 4 <= a.N) {
        if constexpr (EPI == MX_EPI_RESIDUAL) {
          float g[4];
          load_row<bf16_t, 4>(rr + n, g);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] += g[i];
        }
        *reinterpret_cast<uint2*>(yr + n) = make_uint2(bf16_pack2(f[0], f[1]), bf16_pack2(f[2], f[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n + i >= a.N) break;
          if constexpr (EPI == MX_EPI_RESIDUAL) f[i] += to_f32(rr[n + i]);
          yr[n + i] = bf16_from(f[i]);
        }
      }
    }
  }
}

template <bool BOTH, int MT, int NT>
int launch_tile(GemmArgs a, int epilogue, hipStream_t st) {
  using G = GemmTile<BOTH, MT, NT>;
  a.tm = (a.M + G::BM - 1) / G::BM;
  a.tn = (a.N + G::BN - 1) / G::BN;
  const dim3 grid((unsigned)(a.tm * a.tn)), blk(kGemmThreads);
  switch (epilogue) {
    case MX_EPI_NONE:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, MX_EPI_NONE>), grid, blk, G::LDS, st, a);
      break;
    case MX_EPI_GELU:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, MX_EPI_GELU>), grid, blk, G::LDS, st, a);
      break;
    default:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, MX_EPI_RESIDUAL>), grid, blk, G::LDS, st, a);
      break;
  }
  return check_launch("mx4_gemm_kernel");
}

template <bool BOTH>
int launch_gemm(GemmArgs a, int epilogue, hipStream_t st) {
  // offsets inside a tile and tile counts are 32-bit
  if (a.xb * 256 > 0xffffffffLL || (int64_t)a.Kp * 128 > 0xffffffffLL ||
      (int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128) > 0x7fffffffLL) {
    set_error("mx4 product: too large (rows of X of at most 16 MiB apart)");
    return TA_ERR_UNSUPPORTED;
  }
  a.vec = a.ldy % 4 == 0 && (uintptr_t)a.Y % 8 == 0 && (a.R == nullptr || (a.ldr % 4 == 0 && (uintptr_t)a.R % 8 == 0));
  const int64_t big = (int64_t)((a.M + 255) / 256) * ((a.N + 255) / 256);
  if (big * 4 >= (int64_t)device_cus() * 3) return launch_tile<BOTH, 8, 4>(a, epilogue, st);
  return launch_tile<BOTH, 4, 2>(a, epilogue, st);
}

}  // namespace

int mx4_gemm_bf16(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy, const void* R,
                  int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st) {
  GemmArgs a{(const char*)X, ldx * 2, nullptr, (const char*)Wp, (const uint32_t*)Ws, (bf16_t*)Y, ldy, (const bf16_t*)R,
             ldr, M, N, K, mx4_padded(K), 0, 0, 0};
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
  GemmArgs a{(const char*)Xp, mx4_padded(K) / 2, (const uint32_t*)Xs, (const char*)Wp, (const uint32_t*)Ws, (bf16_t*)Y,
             ldy, (const bf16_t*)R, ldr, M, N, K, mx4_padded(K), 0, 0, 0};
  return launch_gemm<true>(a, epilogue, (hipStream_t)stream);
}
