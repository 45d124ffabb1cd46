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
// once by a kernel of their own, into the workspace, from where they go straight to the lanes' registers.  The matrix
// instructions take bf16, and a normalised value rounded to it would be as far off as the result's own rounding: it is held
// as two of them, its upper half and what that leaves (2^-16 of the value is lost), and both are multiplied.
//
// 32 x 4096 x 16384 (35.7 MB of weights) takes 12.4 us, 2.9 TB/s; a floor of 6.5 us at a large copy's rate.  What is left is
// the start (the first weights' round trip), X (every workgroup reads all of it from L2 and turns it round in LDS, twice the
// weights' bytes) and the sums of eight wavefronts at the end.  With a LayerNorm in front it takes 15.0 us and the LayerNorm
// 4.3 (12.4 and 3.5 with its rows rounded to bf16, which made the results' error 1.4 times as large): X has twice the bytes and
// instructions.  1 x 1024 x 1024 takes 3.3 us, a launch with one round trip.
#include "mx4.hpp"

namespace ta {

int mx4_gemm_bf16(const void* X, int64_t ldx, int parts, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                  const void* R, int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st);

namespace {

struct RowsArgs {
  const bf16_t* X;       // X_PARTS: 16-byte unit c * M + r is vector c (of 8 values) of row r, the lower halves Kp / 8 * M on
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

// (x - mean) * rstd * g of eight values, each as the upper half of its float32 (a bf16; the sign, exponent and first bits cut
// off, so nothing overflows) and the rest, rounded to bf16 (0 beside an infinity or NaN).
__device__ __forceinline__ void normalised(const uint4& x, const uint4& g, float mean, float rstd, uint4& hi, uint4& lo) {
  const bf16_t* e = reinterpret_cast<const bf16_t*>(&x);
  const bf16_t* ge = reinterpret_cast<const bf16_t*>(&g);
  uint32_t h[4], l[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t b[2];
    float r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float f = (to_f32(e[2 * u + i]) - mean) * rstd * to_f32(ge[2 * u + i]);
      b[i] = __float_as_uint(f) & 0xffff0000u;
      r[i] = fabsf(f) < INFINITY ? f - __uint_as_float(b[i]) : 0.0f;
    }
    h[u] = b[1] | b[0] >> 16;
    l[u] = bf16_pack2(r[0], r[1]);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
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

// Where the products take X from: bf16 rows; bf16 rows normalised on the way; the two halves of normalised rows in memory, in
// the order the lanes take them.
enum { X_ROWS = 0, X_NORM = 1, X_PARTS = 2 };

// MT 16-row tiles of X, CT 16-column tiles.
template <int MT, int CT, int SRC, int EPI>
__global__ __launch_bounds__(kThreads) void mx4_rows_kernel(RowsArgs a, int ny) {
  constexpr bool LN = SRC == X_NORM, PARTS = SRC == X_PARTS;
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
  const char* xbase = reinterpret_cast<const char*>(a.X) + (PARTS ? (int64_t)m0 * 16 : (int64_t)m0 * a.ldx * 2);
  const int64_t vec = (int64_t)a.M * 16;         // PARTS: bytes from a vector of the rows to the next
  uint32_t xo[MT * 4];
#pragma unroll
  for (int t = 0; t < MT * 4; ++t) {
    const int r = PARTS ? t * 16 + li : t * 4 + lg;
    xo[t] = (uint32_t)(m0 + r < a.M ? r : a.M - 1 - m0) * (PARTS ? 16u : (uint32_t)(a.ldx * 2)) + (PARTS ? 0 : li * 16);
  }
  const bool ragged = (a.K & 127) != 0;
  // this wavefront's step i: its tiles of the weights; rows lg, lg + 4, ... of X's slice, vector li of each
  struct Step {
    uint4 x[LN ? 1 : PARTS ? MT * 8 : MT * 4];
    uint4 q[CT];
    uint32_t s;                                  // the tiles' scales, a byte each
  };
  auto load = [&](int i, Step& v) {
    const int st = st0 + i;
    if constexpr (PARTS) {
      const char* xs = xbase + (st * 16 + lg * 4) * vec;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          v.x[(u * MT + m) * 2] = ldg16(xs + u * vec + xo[m]);
          v.x[(u * MT + m) * 2 + 1] = ldg16(xs + (a.Kp / 8 + u) * vec + xo[m]);
        }
    } else if constexpr (!LN) {
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
      if (v * 8 < a.Kp) {
        char* slot = lds + (v / 16) * XB + x_slot(r, v % 16);
        normalised(x[i], g[i], mean, rstd, *reinterpret_cast<uint4*>(slot), *reinterpret_cast<uint4*>(slot + ks * XB));
      }
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
    if constexpr (SRC == X_ROWS) {
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
      constexpr int P = SRC == X_ROWS ? 1 : 2;
      bf16x8_t ax[MT][P];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < P; ++h)
          if constexpr (PARTS) ax[m][h] = __builtin_bit_cast(bf16x8_t, v.x[(u * MT + m) * 2 + h]);
          else ax[m][h] = *reinterpret_cast<const bf16x8_t*>(xs + h * ks * XB + x_slot(m * 16 + li, lg * 4 + u));
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const bf16x8_t bw = mx4_bf16x8(u == 0 ? v.q[c].x : u == 1 ? v.q[c].y : u == 2 ? v.q[c].z : v.q[c].w, sc[c]);
#pragma unroll
        for (int h = 0; h < P; ++h)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ax[m][h], bw, acc[m][c], 0, 0, 0);
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

// LayerNorm of one row per workgroup, from X to Y, as upper and lower halves, zeros from K to Kp: vector c (of 8 values) of
// row r at byte c * vs + r * rs, the lower half's Kp / 8 vectors on.  Up to 16384 values are held in registers, longer rows
// read again.  The mean, then the squares about it.  32 x 4096: 4.3 us, a launch with one read and two joined sums.
__global__ __launch_bounds__(kThreads) void mx4_norm_kernel(RowsArgs a, char* __restrict__ Y, int64_t rs, int64_t vs) {
  __shared__ float s_red[2][kWaves8];
  const int tid = threadIdx.x;
  const bf16_t* xr = a.X + (int64_t)blockIdx.x * a.ldx;
  char* yr = Y + blockIdx.x * rs;
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
  const int np = a.Kp / 8;
  auto store = [&](int v, const uint4& xv, const uint4& gv) {   // (past K both are 0, and so is the result)
    char* o = yr + v * vs;
    normalised(xv, gv, mean, rstd, *reinterpret_cast<uint4*>(o), *reinterpret_cast<uint4*>(o + np * vs));
  };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * kThreads + tid < np) store(i * kThreads + tid, x[i], g[i]);
  for (int v = NV * kThreads + tid; v < np; v += kThreads) {
    uint4 xv = make_uint4(0, 0, 0, 0), gv = xv;
    if (v < nv) {
      xv = ldg16(xr + (int64_t)v * 8);
      gv = ldg16(a.gam + (int64_t)v * 8);
    }
    store(v, xv, gv);
  }
}

// Whether the product runs as workgroups of 32 rows or as tiles of many rows (mx4_gemm.hip).  The former cost about 8.5 us
// at K = 4096 for every compute unit's worth of workgroups (512 x 4096 x 4096: 1024 of them, 36 us; 128 x 16384: 1024, 40 us;
// 256 x 16384: 2048, 72 us), the latter's 128 x 128 tiles 50 us up to two for a unit.  (Measured at that K alone.  Every
// 32 rows read and convert the weights anew, and 128 x 128 tiles leave half the rate: between 65 and about 512 rows both are
// two to three and a half times their floors.)
bool few_rows(int M, int N) { return M <= 64 || (int64_t)((M + 31) / 32) * ((N + 63) / 64) <= 5 * (int64_t)device_cus(); }

// Whether ta_mx4_rows normalises M rows of K values within the product: wherever a workgroup's LDS holds them (32 x 768 x
// 2304: 6.6 us against 3.1 + 3.8 with the kernel of its own, 4 x 1024 x 4096: 6.0 against 3.1 + 3.4; at the most values 4 x
// 1984 x 8192: 8.4 against 3.1 + 4.4, 32 x 1024 x 4096: 7.6 against 3.3 + 4.3, kernels alone: the second launch is not in it).
bool norm_fused(int M, int K) { return M <= 64 && (int64_t)(M <= 16 ? 16 : 32) * mx4_padded(K) <= kFused; }

template <int MT, int CT, int SRC, int EPI>
int launch_one(const RowsArgs& a, hipStream_t st) {
  constexpr int R = MT * 16, COLS = 16 * CT;
  const int x = SRC == X_NORM ? a.Kp / 128 * R * 512 : SRC == X_ROWS ? kWaves8 * R * 256 : 0;
  const int red = kWaves8 * R * (COLS + 1) * 4;
  const int ny = (a.M + R - 1) / R;
  const dim3 grid((unsigned)((a.N + COLS - 1) / COLS * ny)), blk(kThreads);
  hipLaunchKernelGGL((mx4_rows_kernel<MT, CT, SRC, EPI>), grid, blk, x > red ? x : red, st, a, ny);
  return check_launch("mx4_rows_kernel");
}

template <int MT, int CT, int EPI>
int launch_src(const RowsArgs& a, int src, hipStream_t st) {
  switch (src) {
    case X_ROWS: return launch_one<MT, CT, X_ROWS, EPI>(a, st);
    case X_NORM: return launch_one<MT, CT, X_NORM, EPI>(a, st);
    default: return launch_one<MT, CT, X_PARTS, EPI>(a, st);
  }
}

template <int MT, int CT>
int launch_rows(const RowsArgs& a, int src, int epilogue, hipStream_t st) {
  switch (epilogue) {
    case MX_EPI_NONE: return launch_src<MT, CT, MX_EPI_NONE>(a, src, st);
    case MX_EPI_GELU: return launch_src<MT, CT, MX_EPI_GELU>(a, src, st);
    default: return launch_src<MT, CT, MX_EPI_RESIDUAL>(a, src, st);
  }
}

// The widest workgroup (of 16, 32 or 64 columns) that still leaves every compute unit one: X is read once per workgroup.  32
// rows, K = 4096, in the order 16, 32, 64 columns: N = 4096 7.0, 8.0, 9.7 us; 8192 12.8, 9.8, 11.2; 16384 22.8, 16.6, 12.2.
template <int MT>
int pick_rows(const RowsArgs& a, int src, int epilogue, hipStream_t st) {
  const int cus = device_cus(), ny = (a.M + MT * 16 - 1) / (MT * 16);
  if ((int64_t)((a.N + 63) / 64) * ny >= cus) return launch_rows<MT, 4>(a, src, epilogue, st);
  if ((int64_t)((a.N + 31) / 32) * ny >= cus) return launch_rows<MT, 2>(a, src, epilogue, st);
  return launch_rows<MT, 1>(a, src, epilogue, st);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int64_t ta_mx4_rows_workspace_size(int M, int K, int layernorm) {
  if (!layernorm || M <= 0 || K <= 0 || norm_fused(M, K)) return 0;
  const int64_t half = (int64_t)M * K * 2, few = (int64_t)(M < 8 ? M : 8) * mx4_padded(K) * 4;
  return half > few ? half : few;
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
  const bool few = few_rows(M, N);
  if (ln_w != nullptr && !norm_fused(M, K)) {
    const int64_t need = ta_mx4_rows_workspace_size(M, K, 1), row = (int64_t)a.Kp * 4;
    if (ws == nullptr || ws_bytes < need || (uintptr_t)ws % 16) {
      set_error("ta_mx4_rows: workspace missing, too small or not 16-byte aligned");
      return TA_ERR_WORKSPACE;
    }
    // as many rows at a time as the workspace holds (the results do not depend on how many)
    const int fit = ws_bytes / row < M ? (int)(ws_bytes / row) : M;
    for (int64_t m = 0; m < M; m += fit) {
      RowsArgs c = a;
      c.X += m * ldx;
      c.Y += m * ldy;
      if (R != nullptr) c.R += m * ldr;
      c.M = M - m < fit ? (int)(M - m) : fit;
      hipLaunchKernelGGL(mx4_norm_kernel, dim3((unsigned)c.M), dim3(kThreads), 0, st, c, (char*)ws, few ? 16 : row,
                         few ? (int64_t)c.M * 16 : 16);
      int rc = check_launch("mx4_norm_kernel");
      if (rc != TA_OK) return rc;
      c.X = (const bf16_t*)ws;
      if (!few) rc = mx4_gemm_bf16(ws, row / 2, 2, Wp, Ws, c.Y, ldy, c.R, ldr, c.M, N, a.Kp, epilogue, st);
      else rc = M <= 16 ? pick_rows<1>(c, X_PARTS, epilogue, st) : pick_rows<2>(c, X_PARTS, epilogue, st);
      if (rc != TA_OK) return rc;
    }
    return TA_OK;
  }
  if (!few) return mx4_gemm_bf16(X, ldx, 1, Wp, Ws, Y, ldy, R, ldr, M, N, K, epilogue, st);
  const int src = ln_w != nullptr ? X_NORM : X_ROWS;
  return M <= 16 ? pick_rows<1>(a, src, epilogue, st) : pick_rows<2>(a, src, epilogue, st);
}
