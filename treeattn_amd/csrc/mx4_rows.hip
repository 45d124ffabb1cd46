// Few bf16 rows times 4-bit weights (a decode step's products), on the bf16 matrix instructions:
//   Y[M, N] = epilogue(LN(X)[M, K] . W[N, K]^T), M <= 64.
//
// The step is bound by the weights' bytes (17 of 32 a value), so they go straight from memory to the registers that the
// conversion reads: a lane of v_mfma_f32_16x16x32_bf16 takes row lane % 16 of W and 32 consecutive values of it (one
// block, 16 bytes, one scale), and the four instructions over them take eight each.  The order of k inside a block of
// 128 is thus (i, lane / 16, 8): X is read from LDS in the same order.  Dequantised weights are exact in bf16, so the
// product is that of the bf16 rows with the values the 4 bits stand for, summed in float32.
//
// A workgroup of eight wavefronts computes 16 * CT * WN columns: WN wavefronts side by side, 8 / WN of them over K.  X
// passes through LDS in pieces of kPiece values of K (normalised on the way in when there is a LayerNorm); the weights
// of the next piece are requested before a piece is multiplied.  The partial sums of the wavefronts over K are added in
// LDS in wavefront order.
#include "mx4.hpp"

namespace ta {

int mx4_gemm_bf16(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy, const void* R,
                  int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st);

namespace {

struct RowsArgs {
  const bf16_t* X;
  int64_t ldx;
  const uint4* W;        // blocks of 32: row n's at W + n * (Kp / 32)
  const uint32_t* S;     // four scale bytes each: row n's at S + n * (Kp / 128)
  bf16_t* Y;
  int64_t ldy;
  const bf16_t* R;
  int64_t ldr;
  const bf16_t* gam;
  float eps;
  int M, N, K, Kp;
};

constexpr int kThreads = 512;
constexpr int kWaves8 = 8;

// MT 16-row tiles of X, CT 16-column tiles per wavefront, WN wavefronts side by side; PC: steps of 128 of K per piece
// and wavefront.
template <int MT, int CT, int WN, int PC, bool LN, int EPI>
__global__ __launch_bounds__(kThreads) void mx4_rows_kernel(RowsArgs a) {
  constexpr int WK = kWaves8 / WN;
  constexpr int kPiece = 128 * PC * WK;          // of K
  constexpr int RS = kPiece + 8;                 // LDS row stride in elements: 16 bytes more, off the banks
  constexpr int R = MT * 16;
  constexpr int COLS = 16 * CT * WN;
  extern __shared__ __align__(16) char lds[];
  bf16_t* xs = reinterpret_cast<bf16_t*>(lds);   // [R][RS]
  float* stat = reinterpret_cast<float*>(lds + (size_t)R * RS * 2);   // mean, rstd of each row
  const int tid = threadIdx.x, lane = lane_id(), w = wave_id();
  const int wn = w % WN, wk = w / WN;
  const int li = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * COLS + wn * 16 * CT;
  const int kb = a.Kp / 32, ks = a.Kp / 128;     // blocks, steps of a row

  const uint4* wp[CT];
  const uint32_t* sp[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int n = n0 + c * 16 + li;
    const int nc = n < a.N ? n : a.N - 1;        // columns past the last repeat it and are not stored
    wp[c] = a.W + (int64_t)nc * kb + lg;
    sp[c] = a.S + (int64_t)nc * ks;
  }
  struct Wt {
    uint4 q[PC][CT];
    uint32_t s[PC][CT];
  };
  // the weights of a piece for this wavefront (steps past K repeat the last one; its X is zero)
  auto load_w = [&](int piece, Wt& x) {
#pragma unroll
    for (int i = 0; i < PC; ++i) {
      int st = (piece * PC + i) * WK + wk;
      st = st < ks ? st : ks - 1;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        x.q[i][c] = ldg16(wp[c] + st * 4);
        x.s[i][c] = sp[c][st];
      }
    }
  };
  Wt cur;
  load_w(0, cur);

  if constexpr (LN) {
    // a row's mean and variance by one wavefront, in two passes over values it holds or reads again
    for (int r = w; r < R; r += kWaves8) {
      const bf16_t* xr = a.X + (int64_t)(r < a.M ? r : 0) * a.ldx;
      float s = 0.0f;
      for (int k = lane * 8; k < a.K; k += kWave * 8) {
        float f[8];
        load_row_g<bf16_t, 8>(xr + k, f);
#pragma unroll
        for (int u = 0; u < 8; ++u) s += f[u];
      }
      const float mean = wave_sum(s) / (float)a.K;
      float v = 0.0f;
      for (int k = lane * 8; k < a.K; k += kWave * 8) {
        float f[8];
        load_row_g<bf16_t, 8>(xr + k, f);
#pragma unroll
        for (int u = 0; u < 8; ++u) v += (f[u] - mean) * (f[u] - mean);
      }
      v = wave_sum(v) / (float)a.K;
      if (lane == 0) {
        stat[2 * r] = mean;
        stat[2 * r + 1] = rsqrtf(v + a.eps);
      }
    }
    __syncthreads();
  }

  f32x4_t acc[MT][CT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const int pieces = (a.K + kPiece - 1) / kPiece;
  constexpr int VR = kPiece / 8;                  // vectors of a row
  constexpr int VT = (R * VR + kThreads - 1) / kThreads;
  for (int p = 0; p < pieces; ++p) {
    // X's piece, vector i of it by thread i mod 512
    uint4 xv[VT];
#pragma unroll
    for (int j = 0; j < VT; ++j) {
      const int i = j * kThreads + tid;
      const int r = i / VR, k = p * kPiece + (i % VR) * 8;
      xv[j] = make_uint4(0, 0, 0, 0);
      if (i < R * VR && r < a.M && k < a.K) xv[j] = ldg16(a.X + (int64_t)r * a.ldx + k);
    }
    if (p > 0) __syncthreads();                   // the previous piece has been multiplied
#pragma unroll
    for (int j = 0; j < VT; ++j) {
      const int i = j * kThreads + tid;
      if (i < R * VR) {
        const int r = i / VR, kk = (i % VR) * 8;
        uint4 o = xv[j];
        if constexpr (LN) {
          const int k = p * kPiece + kk;
          if (k < a.K) {
            float f[8], gm[8];
            const bf16_t* e = reinterpret_cast<const bf16_t*>(&xv[j]);
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u] = to_f32(e[u]);
            load_row_g<bf16_t, 8>(a.gam + k, gm);
            const float mean = stat[2 * r], rstd = stat[2 * r + 1];
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u] = (f[u] - mean) * rstd * gm[u];
            o = make_uint4(bf16_pack2(f[0], f[1]), bf16_pack2(f[2], f[3]), bf16_pack2(f[4], f[5]),
                           bf16_pack2(f[6], f[7]));
            if (r >= a.M) o = make_uint4(0, 0, 0, 0);
          }
        }
        *reinterpret_cast<uint4*>(xs + r * RS + kk) = o;
      }
    }
    __syncthreads();
    Wt nxt;
    load_w(p + 1 < pieces ? p + 1 : p, nxt);
#pragma unroll
    for (int i = 0; i < PC; ++i) {
      const int k0 = (i * WK + wk) * 128 + lg * 32;
      float sc[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) sc[c] = mx4_scale((cur.s[i][c] >> (8 * lg)) & 255u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bf16x8_t bw[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const uint32_t q = u == 0 ? cur.q[i][c].x : u == 1 ? cur.q[i][c].y : u == 2 ? cur.q[i][c].z : cur.q[i][c].w;
          bw[c] = mx4_bf16x8(q, sc[c]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const bf16x8_t ax = *reinterpret_cast<const bf16x8_t*>(xs + (m * 16 + li) * RS + k0 + u * 8);
#pragma unroll
          for (int c = 0; c < CT; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ax, bw[c], acc[m][c], 0, 0, 0);
        }
      }
    }
    cur = nxt;
  }

  // sums over the wavefronts along K, then the epilogue: element (row, col) of a tile is register row % 4 of lane
  // (row / 4) * 16 + col
  float* red = reinterpret_cast<float*>(lds);     // [WK][R][COLS + 1]
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[(wk * R + m * 16 + lg * 4 + i) * (COLS + 1) + wn * 16 * CT + c * 16 + li] = acc[m][c][i];
  __syncthreads();
  for (int i = tid; i < R * COLS; i += kThreads) {
    const int r = i / COLS, cc = i % COLS;
    const int n = blockIdx.x * COLS + cc;
    if (r >= a.M || n >= a.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < WK; ++k) s += red[(k * R + r) * (COLS + 1) + cc];
    if constexpr (EPI == MX_EPI_GELU) s = mx4_gelu(s);
    if constexpr (EPI == MX_EPI_RESIDUAL) s += to_f32(a.R[(int64_t)r * a.ldr + n]);
    a.Y[(int64_t)r * a.ldy + n] = bf16_from(s);
  }
}

template <int MT, int CT, int WN, int PC>
int launch_rows(const RowsArgs& a, int epilogue, hipStream_t st) {
  constexpr int WK = kWaves8 / WN, R = MT * 16, COLS = 16 * CT * WN;
  const size_t x = (size_t)R * (128 * PC * WK + 8) * 2 + R * 8;
  const size_t red = (size_t)WK * R * (COLS + 1) * 4;
  const size_t lds = x > red ? x : red;
  const dim3 grid((a.N + COLS - 1) / COLS), blk(kThreads);
#define TA_MXR(L, E) hipLaunchKernelGGL((mx4_rows_kernel<MT, CT, WN, PC, L, E>), grid, blk, lds, st, a)
#define TA_MXL(E)                      \
  if (a.gam != nullptr) TA_MXR(true, E); \
  else TA_MXR(false, E)
  switch (epilogue) {
    case MX_EPI_NONE: TA_MXL(MX_EPI_NONE); break;
    case MX_EPI_GELU: TA_MXL(MX_EPI_GELU); break;
    default: TA_MXL(MX_EPI_RESIDUAL); break;
  }
#undef TA_MXL
#undef TA_MXR
  return check_launch("mx4_rows_kernel");
}

// 64 columns per workgroup where that still leaves every compute unit one, else 16 (32 for more than 32 rows, whose X
// would not fit the LDS of a workgroup with eight wavefronts over K).
template <int MT>
int pick_rows(const RowsArgs& a, int epilogue, hipStream_t st) {
  if ((a.N + 63) / 64 >= device_cus()) return launch_rows<MT, 2, 2, MT == 4 ? 1 : 2>(a, epilogue, st);
  return launch_rows<MT, 1, MT == 4 ? 2 : 1, 1>(a, epilogue, st);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_mx4_rows(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                           const void* R, int64_t ldr, const void* ln_w, float ln_eps, int M, int N, int K,
                           int epilogue, void* stream) {
  if (M < 0 || N < 1 || K < 32 || K % 32 || K > 0x7fffff00 || (M > 1 && (ldx < K || ldy < N)) || epilogue < 0 ||
      epilogue > 2 || (epilogue == MX_EPI_RESIDUAL && (R == nullptr || (M > 1 && ldr < N)))) {
    set_error("ta_mx4_rows: bad sizes (K a multiple of 32; a residual needs its rows)");
    return TA_ERR_ARG;
  }
  if (M == 0) return TA_OK;
  if (X == nullptr || Wp == nullptr || Ws == nullptr || Y == nullptr || ((uintptr_t)X | (uintptr_t)Wp) % 16 ||
      (uintptr_t)Ws % 4 || (ldx * 2) % 16 || (uintptr_t)ln_w % 16 || (uintptr_t)Y % 2) {
    set_error("ta_mx4_rows: X, the packed weights and the LayerNorm weight must be 16-byte aligned with X's row stride "
              "a multiple of 8, the scales 4-byte aligned");
    return TA_ERR_ARG;
  }
  if (ln_w != nullptr && M > 64) {
    set_error("ta_mx4_rows: the LayerNorm prologue takes at most 64 rows");
    return TA_ERR_UNSUPPORTED;
  }
  hipStream_t st = (hipStream_t)stream;
  if (M > 64) return mx4_gemm_bf16(X, ldx, Wp, Ws, Y, ldy, R, ldr, M, N, K, epilogue, st);
  RowsArgs a{(const bf16_t*)X, ldx, (const uint4*)Wp, (const uint32_t*)Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr,
             (const bf16_t*)ln_w, ln_eps, M, N, K, mx4_padded(K)};
  if (M <= 16) return pick_rows<1>(a, epilogue, st);
  if (M <= 32) return pick_rows<2>(a, epilogue, st);
  return pick_rows<4>(a, epilogue, st);
}
