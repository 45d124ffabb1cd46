// Few bf16 rows times 4-bit weights (a decode step's products), on the bf16 matrix instructions:
//   Y[M, N] = epilogue(LN(X)[M, K] . W[N, K]^T).
//
// The step is bound by the weights' bytes (17 of 32 a value), so they go straight from memory to the registers that the
// conversion reads, a tile of 16 columns and 128 of K a load: a lane of v_mfma_f32_16x16x32_bf16 takes one block (16 bytes,
// one scale) of one column, and the four instructions over the tile take eight values of it each.  The order of k inside a block of
// 128 is thus (i, lane / 16, 8): X is read from LDS in the same order.  Dequantised weights are exact in bf16, so the
// product is that of the bf16 rows with the values the 4 bits stand for, summed in float32.
//
// A workgroup of eight wavefronts computes 16 * CT columns of up to 32 rows, each wavefront a run of steps of 128 of K.
// Each value of X is thus used by one wavefront of the workgroup: it reads the step's slice of X by rows and turns it round
// in LDS of its own, without a barrier.  The slices and weights of the next steps are in flight in registers meanwhile;
// loads return in order, so they are issued in the order they are used.  The wavefronts' partial sums are added in LDS in
// wavefront order.
//
// A LayerNorm of short rows (kFused values in all) happens on the way: the workgroup reads X once, 16 or 32 lanes a row,
// and leaves it normalised in LDS for its wavefronts.  Every workgroup does that for itself, so longer rows are normalised
// once by a kernel of their own, into the workspace.  Either way the normalised rows are rounded to bf16, which the
// matrix instructions take.
//
// 32 x 4096 x 16384 (35.7 MB of weights) takes 12.6 us, 2.9 TB/s, and 3.7 for the LayerNorm in front; a floor of 6.5 us at a
// large copy's rate.  What is left is the start (the first weights' round trip), X (every workgroup reads all of it from L2 and
// turns it round in LDS, twice the weights' bytes) and the sums of eight wavefronts at the end.  1 x 1024 x 1024 takes 3.1
// us, a launch with one round trip.
#include "mx4.hpp"

namespace ta {

int mx4_gemm_bf16(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy, const void* R,
                  int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st);

namespace {

struct RowsArgs {
  const bf16_t* X;
  int64_t ldx;
  const char* W;         // tiles of 1024 bytes
  const uint8_t* S;      // scales, 256 bytes for four tiles one below the other
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
constexpr int kFused = 32768;   // values of X, rows and K rounded up to whole tiles and steps, that a workgroup normalises

// Sum over the G lanes (16 or 32, aligned) of a row.
template <int G>
__device__ __forceinline__ float row_sum(float x) { return group_sum<G>(x); }

// (x - mean) * rstd * g of eight values, as bf16.
__device__ __forceinline__ uint4 normalised(const uint4& x, const uint4& g, float mean, float rstd) {
  const bf16_t* e = reinterpret_cast<const bf16_t*>(&x);
  const bf16_t* ge = reinterpret_cast<const bf16_t*>(&g);
  float f[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) f[u] = (to_f32(e[u]) - mean) * rstd * to_f32(ge[u]);
  return make_uint4(bf16_pack2(f[0], f[1]), bf16_pack2(f[2], f[3]), bf16_pack2(f[4], f[5]), bf16_pack2(f[6], f[7]));
}
__device__ __forceinline__ float sum8(const uint4& x) {
  const bf16_t* e = reinterpret_cast<const bf16_t*>(&x);
  float s = 0.0f;
#pragma unroll
  for (int u = 0; u < 8; ++u) s += to_f32(e[u]);
  return s;
}
__device__ __forceinline__ float squares8(const uint4& x, float mean) {
  const bf16_t* e = reinterpret_cast<const bf16_t*>(&x);
  float q = 0.0f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float d = to_f32(e[u]) - mean;
    q = fmaf(d, d, q);
  }
  return q;
}

// The slot of 16-byte vector c (of 16) of row r of a step's slice of X in LDS.  A 16-byte read is served 16 lanes at a time:
// lanes 0-3 and 12-15 of one group of 16 with lanes 4-11 of the next; the groups read vectors four apart.  With rows 4-7
// turned like 0-3 and rows 8-11 like 12-15 those 16 lanes touch every bank once.
__device__ __forceinline__ int x_slot(int r, int c) { return r * 256 + (c ^ ((r & 3) | ((r >> 3) & 1) * 12)) * 16; }

// MT 16-row tiles of X, CT 16-column tiles; LN: normalised on the way.
template <int MT, int CT, bool LN, int EPI>
__global__ __launch_bounds__(kThreads) void mx4_rows_kernel(RowsArgs a, int ny) {
  constexpr int R = MT * 16;
  constexpr int COLS = 16 * CT;
  constexpr int XB = R * 256;                    // bytes of a step's slice of X
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const int li = lane & 15, lg = lane >> 4;
  const int n0 = (int)(blockIdx.x / ny) * COLS, m0 = (int)(blockIdx.x % ny) * R;
  const int ks = a.Kp / 128;                     // steps of a row: dwords of scales, groups of four blocks
  const int per = (ks + kWaves8 - 1) / kWaves8;
  const int st0 = w * per;                       // this wavefront's steps: st0 .. st0 + mine - 1
  const int mine = ks - st0 < per ? (ks > st0 ? ks - st0 : 0) : per;

  // tiles of columns past the last repeat the last tile, rows of X the last row; they are not stored
  const int last = (a.N - 1) / 16;
  int64_t wt[CT];                                // each tile's first
#pragma unroll
  for (int c = 0; c < CT; ++c) wt[c] = (int64_t)(n0 / 16 + c < last ? n0 / 16 + c : last) * ks;
  const uint8_t* sw = a.S + (int64_t)(n0 / 64) * ks * 256 + lane * 4 + n0 / 16 % 4;
  const char* xbase = reinterpret_cast<const char*>(a.X) + (int64_t)m0 * a.ldx * 2;
  uint32_t xo[MT * 4];
#pragma unroll
  for (int t = 0; t < MT * 4; ++t) {
    const int r = t * 4 + lg;
    xo[t] = (uint32_t)(m0 + r < a.M ? r : a.M - 1 - m0) * (uint32_t)(a.ldx * 2) + li * 16;
  }
  const bool ragged = (a.K & 127) != 0;
  // this wavefront's step i: its tiles of the weights; rows lg, lg + 4, ... of X's slice, vector li of each
  struct Step {
    uint4 x[LN ? 1 : MT * 4];
    uint4 q[CT];
    uint32_t s;                                  // the tiles' scales, a byte each
  };
  auto load = [&](int i, Step& v) {
    const int st = st0 + i;
    if constexpr (!LN) {
      const char* xs = xbase + (int64_t)st * 256;
      if (ragged && st == ks - 1) {              // what lies past K is zero
        const bool in = st * 128 + li * 8 < a.K;
#pragma unroll
        for (int t = 0; t < MT * 4; ++t) {
          v.x[t] = ldg16(in ? xs + xo[t] : xbase + xo[t] - li * 16);
          if (!in) v.x[t] = make_uint4(0, 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int t = 0; t < MT * 4; ++t) v.x[t] = ldg16(xs + xo[t]);
      }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) v.q[c] = ldg16(a.W + (wt[c] + st) * 1024 + lane * 16);
    const uint8_t* ss = sw + (int64_t)st * 256;
    v.s = CT == 4 ? *reinterpret_cast<const uint32_t*>(ss) : CT == 2 ? *reinterpret_cast<const uint16_t*>(ss) : *ss;
  };

  Step va, vb;
  if constexpr (LN) {
    // row r of the workgroup's by G lanes, eight vectors each at most
    constexpr int G = kThreads / R, NV = kFused / R / 8 / G;
    const int r = tid / G, j = tid % G;
    const bf16_t* xr = a.X + (int64_t)(m0 + r < a.M ? m0 + r : a.M - 1) * a.ldx;
    uint4 x[NV], g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * G + j) * 8;
      x[i] = g[i] = make_uint4(0, 0, 0, 0);
      if (k < a.K) {
        x[i] = ldg16(xr + k);
        g[i] = ldg16(a.gam + k);
      }
    }
    if (mine > 0) load(0, va);
    if (mine > 1) load(1, vb);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += sum8(x[i]);
    const float mean = row_sum<G>(s) / (float)a.K;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * G + j) * 8 < a.K) q += squares8(x[i], mean);
    const float rstd = rsqrtf(row_sum<G>(q) / (float)a.K + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = i * G + j;                   // vector of the row (past K: weight 0, value 0)
      if (v * 8 < a.Kp) *reinterpret_cast<uint4*>(lds + (v / 16) * XB + x_slot(r, v % 16)) = normalised(x[i], g[i], mean, rstd);
    }
  } else {
    if (mine > 0) load(0, va);
    if (mine > 1) load(1, vb);
  }
  if constexpr (LN) lds_barrier();

  f32x4_t acc[MT][CT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto multiply = [&](int i, Step& v) {
    const char* xs = lds + (LN ? st0 + i : w) * XB;
    if constexpr (!LN) {
      wave_sync();                               // the previous step's slice has been read
#pragma unroll
      for (int t = 0; t < MT * 4; ++t) *reinterpret_cast<uint4*>(lds + w * XB + x_slot(t * 4 + lg, li)) = v.x[t];
      wave_sync();
    }
    float sc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) sc[c] = mx4_scale_of(v.s, c);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8_t ax[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) ax[m] = *reinterpret_cast<const bf16x8_t*>(xs + x_slot(m * 16 + li, lg * 4 + u));
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const bf16x8_t bw = mx4_bf16x8(u == 0 ? v.q[c].x : u == 1 ? v.q[c].y : u == 2 ? v.q[c].z : v.q[c].w, sc[c]);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ax[m], bw, acc[m][c], 0, 0, 0);
      }
    }
    if (i + 2 < mine) load(i + 2, v);
  };
#pragma unroll 1
  for (int i = 0; i < mine; i += 2) {
    multiply(i, va);
    if (i + 1 < mine) multiply(i + 1, vb);
  }

  // sums over the wavefronts, then the epilogue: element (row, col) of a tile is register row % 4 of lane
  // (row / 4) * 16 + col
  float* red = reinterpret_cast<float*>(lds);     // [8][R][COLS + 1]
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[(w * R + m * 16 + lg * 4 + i) * (COLS + 1) + c * 16 + li] = acc[m][c][i];
  __syncthreads();
  for (int i = tid; i < R * COLS; i += kThreads) {
    const int r = i / COLS, cc = i % COLS;
    const int n = n0 + cc;
    if (m0 + r >= a.M || n >= a.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves8; ++k) s += red[(k * R + r) * (COLS + 1) + cc];
    if constexpr (EPI == MX_EPI_GELU) s = mx4_gelu(s);
    if constexpr (EPI == MX_EPI_RESIDUAL) s += to_f32(a.R[(int64_t)(m0 + r) * a.ldr + n]);
    a.Y[(int64_t)(m0 + r) * a.ldy + n] = bf16_from(s);
  }
}

// LayerNorm of one row per workgroup, from X to Y (rows of K, contiguous); up to 16384 values are held in registers, longer
// rows read again.  The mean, then the squares about it.  32 x 4096: 3.7 us, a launch with one read and two joined sums.
__global__ __launch_bounds__(kThreads) void mx4_norm_kernel(RowsArgs a, bf16_t* __restrict__ Y) {
  __shared__ float s_red[2][kWaves8];
  const int tid = threadIdx.x;
  const bf16_t* xr = a.X + (int64_t)blockIdx.x * a.ldx;
  bf16_t* yr = Y + (int64_t)blockIdx.x * a.K;
  const int nv = a.K / 8;
  auto total = [&](float x, int which) {
    x = group_sum<64>(x);
    if (lane_id() == 0) s_red[which][wave_id()] = x;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves8; ++i) t += s_red[which][i];
    return t;
  };
  constexpr int NV = 4;
  uint4 x[NV], g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * kThreads + tid;
    x[i] = g[i] = make_uint4(0, 0, 0, 0);
    if (v < nv) {
      x[i] = ldg16(xr + v * 8);
      g[i] = ldg16(a.gam + v * 8);
    }
  }
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) s += sum8(x[i]);
  for (int v = NV * kThreads + tid; v < nv; v += kThreads) s += sum8(ldg16(xr + (int64_t)v * 8));
  const float mean = total(s, 0) / (float)a.K;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * kThreads + tid < nv) q += squares8(x[i], mean);
  for (int v = NV * kThreads + tid; v < nv; v += kThreads) q += squares8(ldg16(xr + (int64_t)v * 8), mean);
  const float rstd = rsqrtf(total(q, 1) / (float)a.K + a.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = i * kThreads + tid;
    if (v < nv) *reinterpret_cast<uint4*>(yr + v * 8) = normalised(x[i], g[i], mean, rstd);
  }
  for (int v = NV * kThreads + tid; v < nv; v += kThreads)
    *reinterpret_cast<uint4*>(yr + (int64_t)v * 8) =
        normalised(ldg16(xr + (int64_t)v * 8), ldg16(a.gam + (int64_t)v * 8), mean, rstd);
}

// Whether the product runs as workgroups of 32 rows or as tiles of many rows (mx4_gemm.hip).  The former cost about 8.5 us
// at K = 4096 for every compute unit's worth of workgroups (512 x 4096 x 4096: 1024 of them, 36 us; 128 x 16384: 1024, 42 us;
// 256 x 16384: 2048, 72 us), the latter's 128 x 128 tiles 50 us up to two for a unit.
bool few_rows(int M, int N) { return M <= 64 || (int64_t)((M + 31) / 32) * ((N + 63) / 64) <= 5 * (int64_t)device_cus(); }

// Whether ta_mx4_rows normalises M rows of K values within the product: wherever a workgroup's LDS holds them (32 x 768 x
// 2304: 5.6 us against 3.3 + 3.6 with the kernel of its own, 4 x 1024 x 4096: 5.4 against 2.8 + 3.2).
bool norm_fused(int M, int K) { return M <= 64 && (int64_t)(M <= 16 ? 16 : 32) * mx4_padded(K) <= kFused; }

template <int MT, int CT, bool LN, int EPI>
int launch_one(const RowsArgs& a, hipStream_t st) {
  constexpr int R = MT * 16, COLS = 16 * CT;
  constexpr int x = LN ? kFused * 2 : kWaves8 * R * 256, red = kWaves8 * R * (COLS + 1) * 4;
  const int ny = (a.M + R - 1) / R;
  const dim3 grid((unsigned)((a.N + COLS - 1) / COLS * ny)), blk(kThreads);
  hipLaunchKernelGGL((mx4_rows_kernel<MT, CT, LN, EPI>), grid, blk, x > red ? x : red, st, a, ny);
  return check_launch("mx4_rows_kernel");
}

template <int MT, int CT>
int launch_rows(const RowsArgs& a, int epilogue, hipStream_t st) {
  const bool ln = a.gam != nullptr;
  switch (epilogue) {
    case MX_EPI_NONE: return ln ? launch_one<MT, CT, true, MX_EPI_NONE>(a, st) : launch_one<MT, CT, false, MX_EPI_NONE>(a, st);
    case MX_EPI_GELU: return ln ? launch_one<MT, CT, true, MX_EPI_GELU>(a, st) : launch_one<MT, CT, false, MX_EPI_GELU>(a, st);
    default:
      return ln ? launch_one<MT, CT, true, MX_EPI_RESIDUAL>(a, st) : launch_one<MT, CT, false, MX_EPI_RESIDUAL>(a, st);
  }
}

// The widest workgroup (of 16, 32 or 64 columns) that still leaves every compute unit one: X is read once per workgroup.  32
// rows, K = 4096, in the order 16, 32, 64 columns: N = 4096 7.0, 8.0, 9.7 us; 8192 12.8, 9.8, 11.2; 16384 22.8, 16.6, 12.2.
template <int MT>
int pick_rows(const RowsArgs& a, int epilogue, hipStream_t st) {
  const int cus = device_cus(), ny = (a.M + MT * 16 - 1) / (MT * 16);
  if ((int64_t)((a.N + 63) / 64) * ny >= cus) return launch_rows<MT, 4>(a, epilogue, st);
  if ((int64_t)((a.N + 31) / 32) * ny >= cus) return launch_rows<MT, 2>(a, epilogue, st);
  return launch_rows<MT, 1>(a, epilogue, st);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int64_t ta_mx4_rows_workspace_size(int M, int K, int layernorm) {
  return !layernorm || M <= 0 || K <= 0 || norm_fused(M, K) ? 0 : (int64_t)M * K * 2;
}

extern "C" int ta_mx4_rows(const void* X, int64_t ldx, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                           const void* R, int64_t ldr, const void* ln_w, float ln_eps, int M, int N, int K,
                           int epilogue, void* ws, int64_t ws_bytes, void* stream) {
  if (M < 0 || M > 0x7fffff00 || N < 1 || N > 0x7fffff00 || K < 32 || K % 32 || K > 0x7fffff00 || (M > 1 && (ldx < K || ldy < N)) || epilogue < 0 ||
      epilogue > 2 || (epilogue == MX_EPI_RESIDUAL && (R == nullptr || (M > 1 && ldr < N)))) {
    set_error("ta_mx4_rows: bad sizes (K a multiple of 32; a residual needs its rows)");
    return TA_ERR_ARG;
  }
  if (M == 0) return TA_OK;
  if (M > 1 && ldx > (1 << 25)) {
    set_error("ta_mx4_rows: rows of X of at most 2^25 elements apart");
    return TA_ERR_UNSUPPORTED;
  }
  if (X == nullptr || Wp == nullptr || Ws == nullptr || Y == nullptr || ((uintptr_t)X | (uintptr_t)Wp) % 16 ||
      (uintptr_t)Ws % 4 || (ldx * 2) % 16 || (uintptr_t)ln_w % 16 || (uintptr_t)Y % 2) {
    set_error("ta_mx4_rows: X, the packed weights and the LayerNorm weight must be 16-byte aligned with X's row stride "
              "a multiple of 8, the scales 4-byte aligned");
    return TA_ERR_ARG;
  }
  hipStream_t st = (hipStream_t)stream;
  RowsArgs a{(const bf16_t*)X, ldx, (const char*)Wp, Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr,
             (const bf16_t*)ln_w, ln_eps, M, N, K, mx4_padded(K)};
  if (ln_w != nullptr && !norm_fused(M, K)) {
    const int64_t need = ta_mx4_rows_workspace_size(M, K, 1);
    if (ws == nullptr || ws_bytes < need || (uintptr_t)ws % 16) {
      set_error("ta_mx4_rows: workspace missing, too small or not 16-byte aligned");
      return TA_ERR_WORKSPACE;
    }
    hipLaunchKernelGGL(mx4_norm_kernel, dim3((unsigned)M), dim3(kThreads), 0, st, a, (bf16_t*)ws);
    const int rc = check_launch("mx4_norm_kernel");
    if (rc != TA_OK) return rc;
    a.X = (const bf16_t*)ws;
    a.ldx = K;
    a.gam = nullptr;
  }
  if (!few_rows(M, N)) return mx4_gemm_bf16(a.X, a.ldx, Wp, Ws, Y, ldy, R, ldr, M, N, K, epilogue, st);
  return M <= 16 ? pick_rows<1>(a, epilogue, st) : pick_rows<2>(a, epilogue, st);
}
