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

// Slot of 16-byte vector c of row r in an LDS array of rows of eight.  A 16-byte read is served 16 lanes at a time: lanes
// 0-3 and 12-15 of one group of 16 with lanes 4-11 of the next; the groups read vectors two apart of rows that lie two to
// a line of banks.  With this turn those 16 lanes touch every bank once.
__device__ __forceinline__ int turn8(int r) { return ((r >> 1) & 1) | ((r >> 3) & 1) * 6; }
__device__ __forceinline__ int slot8(int r, int c) { return r * 8 + (c ^ turn8(r)); }
// Slot of vector c of row r in an array of rows of two, read in halves.
__device__ __forceinline__ int slot2(int r, int c) { return r * 2 + (c ^ ((r >> 3) & 1)); }

// Copies of 16 or 4 bytes a lane, from a uniform base plus a lane's byte offset (or a lane's own address) to consecutive
// places in LDS.  Written as instructions because the compiler waits for every such copy before the next read of LDS, also
// of another buffer: here copies are in flight while LDS is read, and are waited for by count.  They have no result
// registers, and their operands are read when they issue.
__device__ __forceinline__ void copy16(const void* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(off),
               "s"(base)
               : "memory");
}
__device__ __forceinline__ void copy16(const void* src, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(src)
               : "memory");
}
__device__ __forceinline__ void copy4(const void* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(off),
               "s"(base)
               : "memory");
}
__device__ __forceinline__ void copy4(const void* src, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(src)
               : "memory");
}

// 32 codes as the instruction's operand (which reads its first four registers for 4-bit values).
__device__ __forceinline__ i32x8_t codes(const uint4& q) {
  return i32x8_t{(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
}

template <bool BOTH, int MT, int NT>
struct GemmTile {
  static constexpr int BM = 32 * MT, BN = 64 * NT;
  static constexpr int STEP = BOTH ? 256 : 64;                // of K
  static constexpr int XB = BM * 128;                         // LDS bytes of X a step
  static constexpr int WB = BOTH ? BN * 128 : BN * 32;        // of W
  static constexpr int SB = BOTH ? (BM + BN) * 8 : BN * 4;    // of scales (bf16 X: of two steps)
  static constexpr int BUFS = BOTH ? 2 : 3;                   // steps in LDS
  static constexpr int LDS = BUFS * (XB + WB) + 2 * SB;
};

template <bool BOTH, int MT, int NT, int EPI>
__global__ __launch_bounds__(kGemmThreads) void mx4_gemm_kernel(GemmArgs a) {
  using G = GemmTile<BOTH, MT, NT>;
  constexpr int BM = G::BM, BN = G::BN;
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
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
    xc[i] = (s % 8) ^ turn8(r);
    xo[i] = (uint32_t)(m0 + r < a.M ? r : a.M - 1 - m0) * (uint32_t)a.xb + xc[i] * 16;
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int s = (i * 8 + w) * 64 + lane;
    const int r = BOTH ? s / 8 : s / 2;
    wc[i] = BOTH ? (s % 8) ^ turn8(r) : (s % 2) ^ ((r >> 3) & 1);
    wo[i] = (uint32_t)(n0 + r < a.N ? r : a.N - 1 - n0) * (uint32_t)(a.Kp / 2) + wc[i] * 16;
  }
  const char* xsc = reinterpret_cast<const char*>(a.XS) + (int64_t)m0 * kd * 4;   // scales, from the tile's first row
  const char* wsc = reinterpret_cast<const char*>(a.S) + (int64_t)n0 * kd * 4;
  uint32_t so[NS];
  int sd[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int s = (i * 8 + w) * 64 + lane;
    const int r = BOTH ? (s / 2 < BM ? s / 2 : s / 2 - BM) : s;
    sd[i] = BOTH ? s & 1 : 0;
    const int rr = BOTH && s / 2 < BM ? (m0 + r < a.M ? r : a.M - 1 - m0) : (n0 + r < a.N ? r : a.N - 1 - n0);
    so[i] = (uint32_t)(rr * kd + sd[i]) * 4;
  }
  const bool ragged = BOTH ? (a.Kp & 255) != 0 : (a.K & 63) != 0;

  constexpr int BUFS = G::BUFS;
  auto lx = [&](int buf) { return lds + buf * G::XB; };
  auto lw = [&](int buf) { return lds + BUFS * G::XB + buf * G::WB; };
  auto ls = [&](int buf) { return lds + BUFS * (G::XB + G::WB) + buf * G::SB; };

  auto stage = [&](int s, int buf) {
    const char* xs = xbase + (int64_t)s * 128;
    const char* ws = wbase + (int64_t)s * (BOTH ? 128 : 32);
    if (ragged && s == steps - 1) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const bool in = BOTH ? s * 8 + xc[i] < kd * 4 : s * 64 + xc[i] * 8 < a.K;
        copy16(in ? (const void*)(xs + xo[i]) : (const void*)&kZeros, lx(buf) + (i * 8 + w) * 1024);
      }
      if constexpr (BOTH) {
#pragma unroll
        for (int i = 0; i < NW; ++i)
          copy16(s * 8 + wc[i] < kd * 4 ? (const void*)(ws + wo[i]) : (const void*)&kZeros, lw(buf) + (i * 8 + w) * 1024);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const char* sb = (i * 8 + w) * 32 < BM ? xsc : wsc;
          copy4(s * 2 + sd[i] < kd ? (const void*)(sb + s * 8 + so[i]) : (const void*)&kZeros, ls(buf) + (i * 8 + w) * 256);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NX; ++i) copy16(xs, xo[i], lx(buf) + (i * 8 + w) * 1024);
      if constexpr (BOTH) {
#pragma unroll
        for (int i = 0; i < NW; ++i) copy16(ws, wo[i], lw(buf) + (i * 8 + w) * 1024);
#pragma unroll
        for (int i = 0; i < NS; ++i)
          copy4(((i * 8 + w) * 32 < BM ? xsc : wsc) + s * 8, so[i], ls(buf) + (i * 8 + w) * 256);
      }
    }
    if constexpr (!BOTH) {
      if (w < BN / 32) copy16(ws, wo[0], lw(buf) + w * 1024);
      if ((s & 1) == 0 && w < BN / 64) copy4(wsc + (s >> 1) * 4, so[0], ls((s >> 1) & 1) + w * 256);
    }
  };

  f32x4_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // The operands of row tile m + 1 are read while the instructions of row tile m run.
  auto multiply = [&](int s, int buf) {
    const uint4* x = reinterpret_cast<const uint4*>(lx(buf));
    if constexpr (BOTH) {
      const uint4* wl = reinterpret_cast<const uint4*>(lw(buf));
      const uint16_t* sc = reinterpret_cast<const uint16_t*>(ls(buf));
      i32x8_t wq[2][NT];
      int sw[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int r = wn + c * 16 + li;
        sw[c] = sc[(BM + r) * 4 + lg];
#pragma unroll
        for (int k = 0; k < 2; ++k) wq[k][c] = codes(wl[slot8(r, lg * 2 + k)]);
      }
      i32x8_t xq[2][2];
      int sx[2];
      auto read = [&](int m, int j) {
        const int r = wm + m * 16 + li;
        sx[j] = sc[r * 4 + lg];
#pragma unroll
        for (int k = 0; k < 2; ++k) xq[j][k] = codes(x[slot8(r, lg * 2 + k)]);
      };
      read(0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m + 1 < MT) read(m + 1, (m + 1) & 1);
#pragma unroll
        for (int c = 0; c < NT; ++c)
          acc[m][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wq[0][c], xq[m & 1][0], acc[m][c], 4, 4, 0, sw[c], 0,
                                                                       sx[m & 1]);
#pragma unroll
        for (int c = 0; c < NT; ++c)
          acc[m][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wq[1][c], xq[m & 1][1], acc[m][c], 4, 4, 1, sw[c], 1,
                                                                       sx[m & 1]);
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * NT, 0);
      }
    } else {
      const uint2* wl = reinterpret_cast<const uint2*>(lw(buf));
      const uint8_t* sc = reinterpret_cast<const uint8_t*>(ls((s >> 1) & 1)) + 2 * (s & 1) + (lg >> 1);
      bf16x8_t xv[2][2];
      auto read = [&](int m, int j) {
        const int r = wm + m * 16 + li;
#pragma unroll
        for (int k = 0; k < 2; ++k) xv[j][k] = __builtin_bit_cast(bf16x8_t, x[slot8(r, lg * 2 + k)]);
      };
      uint2 q[NT];
      uint32_t sb[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int r = wn + c * 16 + li;
        q[c] = wl[slot2(r, lg >> 1) * 2 + (lg & 1)];
        sb[c] = sc[r * 4];
      }
      read(0, 0);
      bf16x8_t wv[NT][2];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const float f = mx4_scale(sb[c]);
        wv[c][0] = mx4_bf16x8(q[c].x, f);
        wv[c][1] = mx4_bf16x8(q[c].y, f);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m + 1 < MT) read(m + 1, (m + 1) & 1);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int c = 0; c < NT; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[c][k], xv[m & 1][k], acc[m][c], 0, 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * NT, 0);
      }
    }
  };

  // Step s + BUFS - 1 is requested when step s begins, into the buffer of step s - 1, which everyone has left by then.
  stage(0, 0);
  if (BUFS == 3 && steps > 1) stage(1, 1);
  int buf = 0;
  for (int s = 0; s < steps; ++s) {
    // this wavefront's copies of step s have landed; with three buffers those of step s + 1 may be on their way
    if constexpr (BOTH) {
      wait_vmcnt_n<0>();
    } else {
      const int later = s + 1 < steps ? NX + (w < BN / 32) + ((s & 1) && w < BN / 64) : 0;
      if (later == NX + 2) wait_vmcnt_n<NX + 2>();
      else if (later == NX + 1) wait_vmcnt_n<NX + 1>();
      else if (later == NX) wait_vmcnt_n<NX>();
      else wait_vmcnt_n<0>();
    }
    lds_barrier();       // everyone's have
    const int next = buf == 0 ? BUFS - 1 : buf - 1;
    if (s + BUFS - 1 < steps) stage(s + BUFS - 1, next);
    multiply(s, buf);
    buf = buf == BUFS - 1 ? 0 : buf + 1;
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
