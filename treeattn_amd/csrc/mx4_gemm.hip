// Products with 4-bit weights over many rows: Y[M, N] = epilogue(X[M, K] . W[N, K]^T) with X in bf16 (the weights made
// bf16, exactly, in front of the bf16 matrix instructions) or in 4 bits as well (v_mfma_scale_f32_16x16x128_f8f6f4 on the
// codes and scales as they are).  Sums are float32, the result is rounded once after the epilogue.
//
// A workgroup of eight wavefronts, two along M by four along N, computes a (32 MT) x (64 NT) tile; a wavefront MT x NT
// instruction tiles of it.  K goes through LDS in steps of 128 (both in 4 bits) or 64 (bf16 X), copied there straight from
// memory, the copies of the next BUFS - 1 steps in flight.  Tiles of 4-bit rows are copied and read as they are, lane by
// lane; of bf16 X the rows are, 128 bytes a step, turned so that LDS reads touch every bank once.  The weights are the
// instructions' first operand, so a lane ends with four consecutive columns of one row.
//
// With bf16 X a lane takes half a block of weights a step (k = 16g .. 16g + 15 of the step's 64 for lane group g): eight
// bytes of codes and one scale serve its two instructions.  Rows and tiles past the last repeat it and are not stored; what
// a step has past K is read as zeros.
//
// Bound by the matrix instructions and what feeds them.  Times are medians of kernel traces, calls of several inputs in turn
// (many calls of one input in a row differ by the clock and by what stays in the caches).  bf16 X, 2001 x 2048 x 8192: 58 us,
// 1157 TFLOP/s (a large library product of bf16 matrices 1377 on that card, twenty in a row); the instructions are busy 46 %
// of the time, the rest is the phases' barriers, the conversions and a fixed part (start, first copies, 32 MB of results).  Both
// in 4 bits, 4096 x 4096 x 8192: 74 us, 3.7 PFLOP/s of the 8.5 to 9.6 that the instructions alone reach from registers: about
// 31 us of instructions, 8 of barriers, 15 of the fixed part (67 MB of results) and 20 in which LDS reads, copies and
// instructions hold each other up.  The clock is part of it: fifty such products of one input in a row take 87 us each on
// random values and 66 on zeros.  Four wavefronts of 128 x
// 128, one to a SIMD with the next operands read during a step's instructions (two thirds of the LDS reads, one barrier a
// step), took 82 us.
#include "mx4.hpp"

namespace ta {
namespace {

struct GemmArgs {
  const char* X;         // bf16: rows of xb bytes; 4 bits: tiles
  int64_t xb;
  const uint8_t* XS;     // 4-bit X: its scales
  const char* W;
  const uint8_t* S;
  bf16_t* Y;
  int64_t ldy;
  const bf16_t* R;
  int64_t ldr;
  int M, N, K, ks;       // ks: steps of 128 in a row of W
  int wsteps;            // bf16 X: steps of 64 after which W starts again (X holds its upper and then its lower halves)
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

// Copies of 16 or 4 bytes a lane, from a uniform base plus a lane's byte offset (or a lane's own address) to consecutive
// places in LDS.  Written as instructions because the compiler waits for every such copy before the next read of LDS, also
// of another buffer: here copies are in flight while LDS is read, and are waited for by count.  They have no result
// registers, and their operands are read when they issue.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // (m0 is one of the compiler's own registers, as meant)
__device__ __forceinline__ void copy16(const void* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(off),
               "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void copy16(const void* src, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(src)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(const void* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"((uint32_t)(uintptr_t)(lds_void*)dst), "v"(off),
               "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Workgroups go to the eight XCDs in turn: each XCD takes a contiguous run of tiles, in groups of eight rows of tiles, so
// that what its workgroups share stays in its L2.
__device__ __forceinline__ void tile_of(const GemmArgs& a, int& tm, int& tn) {
  const int T = a.tm * a.tn, id = blockIdx.x, x = id & 7, q = T >> 3, r = T & 7;
  const int t = x * q + (x < r ? x : r) + (id >> 3);
  const int per = 8 * a.tn, g = t / per, gm = a.tm - g * 8 < 8 ? a.tm - g * 8 : 8;
  tm = g * 8 + (t - g * per) % gm;
  tn = (t - g * per) / gm;
}

// The epilogue of a wavefront's MT x NT instruction tiles from row m0 and column n0: element (column n, row m) of a tile is
// register n % 4 of lane (n / 4) * 16 + m.  Rows go through LDS of the wavefront's own (16 of them at a time, 8 bytes more
// apart than they are long) so that they are stored, and the residual read, in whole runs of 16 NT columns.
template <int MT, int NT, int EPI>
__device__ __forceinline__ void store_tile(const GemmArgs& a, const f32x4_t (&acc)[MT][NT], int m0, int n0, int li, int lg,
                                           char* lds) {
  constexpr int RB = NT * 32 + 8;                             // bytes of a row in LDS
  constexpr int LR = NT * 4;                                  // lanes of a row, four columns each
  const int lane = lg * 16 + li;
  const int n = n0 + lane % LR * 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    char* buf = lds + (m & 1) * 16 * RB;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = EPI == MX_EPI_GELU ? mx4_gelu(acc[m][c][i]) : acc[m][c][i];
      if constexpr (EPI == MX_EPI_RESIDUAL) {                 // added before the one rounding: in place, not through LDS
        const int row = m0 + m * 16 + li, nn = n0 + c * 16 + lg * 4;
        if (row < a.M) {
          const bf16_t* rr = a.R + (int64_t)row * a.ldr + nn;
          if (a.vec && nn + 4 <= a.N) {
            float g[4];
            load_row<bf16_t, 4>(rr, g);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] += g[i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (nn + i < a.N) f[i] += to_f32(rr[i]);
          }
        }
      }
      *reinterpret_cast<uint2*>(buf + li * RB + c * 32 + lg * 8) = make_uint2(bf16_pack2(f[0], f[1]), bf16_pack2(f[2], f[3]));
    }
    wave_sync();
#pragma unroll
    for (int j = 0; j < NT; ++j) {                            // 64 / LR rows at a time
      const int r = j * (64 / LR) + lane / LR;
      const int row = m0 + m * 16 + r;
      const uint2 v = *reinterpret_cast<const uint2*>(buf + r * RB + lane % LR * 8);
      if (row < a.M) {
        bf16_t* yr = a.Y + (int64_t)row * a.ldy + n;
        if (a.vec && n + 4 <= a.N) {
          *reinterpret_cast<uint2*>(yr) = v;
        } else {
          const bf16_t* e = reinterpret_cast<const bf16_t*>(&v);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < a.N) yr[i] = e[i];
        }
      }
    }
    wave_sync();
  }
}

// Waits until at most n of this wavefront's copies are on their way (n uniform, up to 24).
__device__ __forceinline__ void wait_copies(int n) {
  switch (n) {
#define TA_WAIT(N) case N: wait_vmcnt_n<N>(); break;
    TA_WAIT(1) TA_WAIT(2) TA_WAIT(3) TA_WAIT(4) TA_WAIT(5) TA_WAIT(6) TA_WAIT(7) TA_WAIT(8) TA_WAIT(9) TA_WAIT(10)
    TA_WAIT(11) TA_WAIT(12) TA_WAIT(13) TA_WAIT(14) TA_WAIT(15) TA_WAIT(16) TA_WAIT(17) TA_WAIT(18) TA_WAIT(19)
    TA_WAIT(20) TA_WAIT(21) TA_WAIT(22) TA_WAIT(23) TA_WAIT(24)
#undef TA_WAIT
    default: wait_vmcnt_n<0>();
  }
}

// 32 codes as the instruction's operand (which reads its first four registers for 4-bit values).
__device__ __forceinline__ i32x8_t codes(const uint4& q) {
  return i32x8_t{(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
}

// The instruction with byte wi of ws and byte xi of xs as scales (the bytes known when unrolled: they are part of it).
__device__ __forceinline__ f32x4_t multiply4(const i32x8_t& w, const i32x8_t& x, const f32x4_t& c, int ws, int wi, int xs,
                                             int xi) {
#define TA_M4(A, B) \
  if (wi == A && xi == B) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, A, ws, B, xs);
  TA_M4(0, 0) TA_M4(0, 1) TA_M4(0, 2) TA_M4(0, 3) TA_M4(1, 0) TA_M4(1, 1) TA_M4(1, 2) TA_M4(1, 3)
  TA_M4(2, 0) TA_M4(2, 1) TA_M4(2, 2) TA_M4(2, 3) TA_M4(3, 0) TA_M4(3, 1) TA_M4(3, 2)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 3, ws, 3, xs);
#undef TA_M4
}

template <bool BOTH, int MT, int NT>
struct GemmTile {
  static constexpr int BM = 32 * MT, BN = 64 * NT;
  static constexpr int XT = BM / 16, WT = BN / 16;            // 16-row tiles
  static constexpr int XB = BOTH ? XT * 1024 : BM * 128;      // LDS bytes of a step: X
  static constexpr int WB = WT * (BOTH ? 1024 : 512);         // W
  static constexpr int SB = (BOTH ? XT + WT : WT) * 64;       // scales (bf16 X: of two steps), 256 of four tiles
  static constexpr int BUFS = BOTH ? 4 : 3;   // (six for MT 4: 256 x 4096 x 16384 54 -> 59 us, one workgroup a unit)
  static constexpr int SBUFS = BOTH ? BUFS : 2;
  static constexpr int LDS = BUFS * (XB + WB) + SBUFS * SB;
};

// PAIRED (MT 8, NT 4): the wavefronts stand two to a SIMD, and the second of each pair (w >= 4) runs half a phase behind the
// first, so that one multiplies (32 instructions, 512 cycles) while the other reads its next operands from LDS, makes bf16
// of its weights and issues copies.  A barrier ends each phase.
template <bool BOTH, int MT, int NT, bool PAIRED, int EPI>
__global__ __launch_bounds__(kGemmThreads) void mx4_gemm_kernel(GemmArgs a) {
  using G = GemmTile<BOTH, MT, NT>;
  constexpr int BM = G::BM, BN = G::BN, XT = G::XT, WT = G::WT, BUFS = G::BUFS;
  constexpr int NX = BOTH ? XT / 8 : BM / 64;                 // copies of X of a wavefront and step
  constexpr int NSC = (BOTH ? XT + WT : WT) / 4;              // wavefronts that copy scales
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const int li = lane & 15, lg = lane >> 4;
  const int wm = (w >> 2) * MT, wn = (w & 3) * NT;            // this wavefront's first tiles
  int m0, n0;
  tile_of(a, m0, n0);
  m0 *= BM;
  n0 *= BN;
  const int steps = BOTH ? a.ks : (a.K + 63) / 64;
  const int lastx = (a.M - 1) / 16 - m0 / 16, lastw = (a.N - 1) / 16 - n0 / 16;

  auto lx = [&](int buf) { return lds + buf * G::XB; };
  auto lw = [&](int buf) { return lds + BUFS * G::XB + buf * G::WB; };
  auto ls = [&](int buf) { return lds + BUFS * (G::XB + G::WB) + buf * G::SB; };

  // what this wavefront copies: uniform bases, and lanes' byte offsets from them
  const int64_t tstep = (int64_t)a.ks * 1024;                 // from a 16-row tile to the next
  const char* xb;
  uint32_t xo[NX];
  int xc[NX];
  if constexpr (BOTH) {
    xb = a.X + (m0 / 16) * tstep;
#pragma unroll
    for (int i = 0; i < NX; ++i) xo[i] = lane * 16;
  } else {
    xb = a.X + (int64_t)m0 * a.xb;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int s = (i * 8 + w) * 64 + lane, r = s / 8;
      xc[i] = (s % 8) ^ turn8(r);
      xo[i] = (uint32_t)(m0 + r < a.M ? r : a.M - 1 - m0) * (uint32_t)a.xb + xc[i] * 16;
    }
  }
  const char* wb = a.W + (n0 / 16) * tstep;
  uint32_t wo = lane * 16;
  if constexpr (!BOTH) {                                      // half tiles 2w and 2w + 1
    const int t = 2 * w + (lane >> 5);
    wo = (uint32_t)(t < lastw ? t : lastw) * (uint32_t)(a.ks * 1024) + (lane & 31) * 16;
  }
  // scales of four tiles: wavefront w's group of them
  const char* sb;
  {
    const bool x = BOTH && w < XT / 4;
    const int g = BOTH && !x ? w - XT / 4 : w, l = (x ? lastx + m0 / 16 : lastw + n0 / 16) / 4 - (x ? m0 : n0) / 64;
    sb = reinterpret_cast<const char*>(x ? a.XS : a.S) + ((int64_t)((x ? m0 : n0) / 64) + (g < l ? g : l)) * a.ks * 256;
  }
  const bool ragged = !BOTH && (a.K & 63) != 0;

  // copy i of step s by this wavefront (i known when unrolled): those of X, of W, of scales
  constexpr int NC = NX + (BOTH ? WT / 8 : 1) + 1;
  auto copy = [&](int s, int buf, int i, bool tail) {
    const int u = !BOTH && s >= a.wsteps ? s - a.wsteps : s;   // step of W
    if (i < NX) {
      if constexpr (BOTH) {
        const int t = i * 8 + w;
        copy16(xb + (t < lastx ? t : lastx) * tstep + (int64_t)s * 1024, xo[i], lx(buf) + t * 1024);
      } else {
        const char* xs = xb + (int64_t)s * 128;
        char* dst = lx(buf) + (i * 8 + w) * 1024;
        if (tail)                                              // what lies past K is zeros
          copy16(s * 64 + xc[i] * 8 < a.K ? (const void*)(xs + xo[i]) : (const void*)&kZeros, dst);
        else
          copy16(xs, xo[i], dst);
      }
    } else if (i < NC - 1) {
      if constexpr (BOTH) {
        const int t = (i - NX) * 8 + w;
        copy16(wb + (t < lastw ? t : lastw) * tstep + (int64_t)s * 1024, wo, lw(buf) + t * 1024);
      } else if (w < WT / 2) {
        copy16(wb + (int64_t)(u >> 1) * 1024 + (u & 1) * 512, wo, lw(buf) + w * 1024);
      }
    } else if (w < NSC) {
      if constexpr (BOTH) copy4(sb + (int64_t)s * 256, lane * 4, ls(buf) + w * 256);
      else if ((s & 1) == 0) copy4(sb + (int64_t)(u >> 1) * 256, lane * 4, ls((s >> 1) % G::SBUFS) + w * 256);
    }
  };
  auto stage = [&](int s, int buf) {
    if (ragged && s == steps - 1) {
#pragma unroll
      for (int i = 0; i < NC; ++i) copy(s, buf, i, true);
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) copy(s, buf, i, false);
    }
  };
  // copies of this wavefront in step s
  auto copies = [&](int s) {
    return BOTH ? NX + WT / 8 + (w < NSC) : NX + (w < WT / 2) + ((s & 1) == 0 && w < NSC);
  };
  // waits for the copies of every issued step before s; the last issued one is `end` - 1
  auto wait = [&](int s, int end) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < BUFS - 1; ++i)
      if (s + i < end) n += copies(s + i);
    wait_copies(n);
  };
  auto phase = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // end of the operands' phase and of the instructions' phase
  auto begin = [&]() {
    if constexpr (PAIRED) {
      phase();
      __builtin_amdgcn_s_setprio(1);
    }
  };
  auto finish = [&]() {
    if constexpr (PAIRED) {
      __builtin_amdgcn_s_setprio(0);
      phase();
    }
  };

  f32x4_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[m][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (int s = 0; s < BUFS - 1; ++s)
    if (s < steps) stage(s, s);
  if constexpr (PAIRED) {
    wait(1, steps < BUFS - 1 ? steps : BUFS - 1);
    phase();
    if (w >= 4) phase();
  }
  int buf = 0;
  for (int s = 0; s < steps; ++s) {
    const int next = buf == 0 ? BUFS - 1 : buf - 1;           // the buffer of step s - 1, which everyone has left
    const int ahead = s + BUFS - 1;
    if constexpr (!PAIRED) {
      wait(s + 1, ahead < steps ? ahead : steps);
      phase();                                                // everyone's copies of step s have landed
      if (ahead < steps) stage(ahead, next);
    }
    if constexpr (BOTH) {
      const uint4* x = reinterpret_cast<const uint4*>(lx(buf)) + wm * 64 + lane;
      const uint4* wl = reinterpret_cast<const uint4*>(lw(buf)) + wn * 64 + lane;
      const int* sx = reinterpret_cast<const int*>(ls(buf)) + wm / 4 * 64 + lane;
      const int sw = reinterpret_cast<const int*>(ls(buf))[(XT + wn) / 4 * 64 + lane] >> (NT < 4 ? wn % 4 * 8 : 0);
      i32x8_t wq[NT], xq[MT];
      int fx[MT / 4];
#pragma unroll
      for (int c = 0; c < NT; ++c) wq[c] = codes(wl[c * 64]);
#pragma unroll
      for (int m = 0; m < MT; ++m) xq[m] = codes(x[m * 64]);
#pragma unroll
      for (int m = 0; m < MT / 4; ++m) fx[m] = sx[m * 64];
      if (PAIRED && s + 1 < steps) wait(s + 2, ahead < steps ? ahead : steps);
      begin();
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
          acc[m][c] = multiply4(wq[c], xq[m], acc[m][c], sw, c, fx[m / 4], m % 4);
        if constexpr (PAIRED) {
          // a copy of step `ahead` between two row tiles' instructions, where issuing it costs nothing (as a phase of its own
          // with the LDS reads it cost 12 of 86 us at 4096 x 4096 x 8192; with bf16 X, whose copies are a smaller part, the
          // same move lost 2 of 57 us at 2001 x 2048 x 8192)
          if (m < NC && ahead < steps) {
            __builtin_amdgcn_sched_barrier(0);
            copy(ahead, next, m, false);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      finish();
    } else {
      const uint4* x = reinterpret_cast<const uint4*>(lx(buf)) + (wm * 16 + li) * 8;
      const uint2* wl = reinterpret_cast<const uint2*>(lw(buf)) + wn * 64 + ((lg >> 1) * 16 + li) * 2 + (lg & 1);
      const uint32_t sw = reinterpret_cast<const uint32_t*>(ls((s >> 1) % G::SBUFS))[wn / 4 * 64 + (2 * (s & 1) + (lg >> 1)) * 16 + li] >>
                          (NT < 4 ? wn % 4 * 8 : 0);
      uint2 q[NT];
      float f[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        q[c] = wl[c * 64];
        f[c] = mx4_scale_of(sw, c);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        bf16x8_t wv[NT], xv[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xv[m] = __builtin_bit_cast(bf16x8_t, x[m * 128 + ((lg * 2 + k) ^ turn8(li))]);
#pragma unroll
        for (int c = 0; c < NT; ++c) wv[c] = mx4_bf16x8(k ? q[c].y : q[c].x, f[c]);
        if constexpr (PAIRED) {
          if (k == 0 && ahead < steps) stage(ahead, next);
          if (k == 1 && s + 1 < steps) wait(s + 2, ahead < steps ? ahead + 1 : steps);
        }
        begin();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int c = 0; c < NT; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[c], xv[m], acc[m][c], 0, 0, 0);
        finish();
      }
    }
    buf = buf == BUFS - 1 ? 0 : buf + 1;
  }
  if (PAIRED && w < 4) phase();
  __syncthreads();                                            // everyone has left the operands' LDS
  store_tile<MT, NT, EPI>(a, acc, m0 + wm * 16, n0 + wn * 16, li, lg, lds + w * 32 * (NT * 32 + 8));
}

template <bool BOTH, int MT, int NT, bool PAIRED>
int launch_tile(GemmArgs a, int epilogue, hipStream_t st) {
  using G = GemmTile<BOTH, MT, NT>;
  a.tm = (a.M + G::BM - 1) / G::BM;
  a.tn = (a.N + G::BN - 1) / G::BN;
  const dim3 grid((unsigned)(a.tm * a.tn)), blk(kGemmThreads);
  switch (epilogue) {
    case MX_EPI_NONE:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, PAIRED, MX_EPI_NONE>), grid, blk, G::LDS, st, a);
      break;
    case MX_EPI_GELU:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, PAIRED, MX_EPI_GELU>), grid, blk, G::LDS, st, a);
      break;
    default:
      hipLaunchKernelGGL((mx4_gemm_kernel<BOTH, MT, NT, PAIRED, MX_EPI_RESIDUAL>), grid, blk, G::LDS, st, a);
      break;
  }
  return check_launch("mx4_gemm_kernel");
}

template <bool BOTH>
int launch_gemm(GemmArgs a, int epilogue, hipStream_t st) {
  // offsets inside a tile and tile counts are 32-bit
  if ((!BOTH && a.xb * 256 > 0xffffffffLL) || a.ks > 65536 ||
      (int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128) > 0x7fffffffLL) {
    set_error("mx4 product: too large (K of at most 8388608, rows of X of at most 16 MiB apart; with a LayerNorm K of at "
              "most 4194304)");
    return TA_ERR_UNSUPPORTED;
  }
  a.vec = a.ldy % 4 == 0 && (uintptr_t)a.Y % 8 == 0 && (a.R == nullptr || (a.ldr % 4 == 0 && (uintptr_t)a.R % 8 == 0));
  // Rounds of tiles over the compute units: one of 256 x 256 tiles takes about three of 128 x 128 (bf16 X, N 8192, K 4096;
  // M 1024: 97 against 70 us, 1536: 101 against 108, 2048: 108 against 140, 2304, whose 288 large tiles are two rounds: 193
  // against 167.  Both in 4 bits: 35 and 27, 36.9 and 37.4, 38.6 and 46.8, 65 and 56 us).  Few rows of 4 bits have no form of
  // their own: 1 to 128 rows x 4096 x 4096 or 16384 take 15 to 16 us, a workgroup's whole walk along K.
  const int64_t cus = device_cus(), rounds = ((int64_t)((a.M + 255) / 256) * ((a.N + 255) / 256) + cus - 1) / cus,
                small = ((int64_t)((a.M + 127) / 128) * ((a.N + 127) / 128) + cus - 1) / cus;
  if (small < 3 * rounds) return launch_tile<BOTH, 4, 2, false>(a, epilogue, st);
  return launch_tile<BOTH, 8, 4, true>(a, epilogue, st);
}

}  // namespace

// parts 2: a row of X is its values' upper halves and then their lower halves, and K a multiple of 128 (so that W starts again
// at a whole tile).
int mx4_gemm_bf16(const void* X, int64_t ldx, int parts, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                  const void* R, int64_t ldr, int M, int N, int K, int epilogue, hipStream_t st) {
  GemmArgs a{(const char*)X, ldx * 2, nullptr, (const char*)Wp, Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr, M, N,
             (int)((int64_t)K * parts), mx4_padded(K) / 128, (K + 63) / 64, 0, 0, 0};
  return launch_gemm<false>(a, epilogue, st);
}

}  // namespace ta

using namespace ta;

extern "C" int ta_mx4_both(const void* Xp, const uint8_t* Xs, const void* Wp, const uint8_t* Ws, void* Y, int64_t ldy,
                           const void* R, int64_t ldr, int M, int N, int K, int epilogue, void* stream) {
  if (M < 0 || M > 0x7fffff00 || N < 1 || N > 0x7fffff00 || K < 1 || K > 0x7fffff00 || (M > 1 && ldy < N) || epilogue < 0 || epilogue > 2 ||
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
  GemmArgs a{(const char*)Xp, 0, Xs, (const char*)Wp, Ws, (bf16_t*)Y, ldy, (const bf16_t*)R, ldr, M, N, K,
             mx4_padded(K) / 128, 0, 0, 0, 0};
  return launch_gemm<true>(a, epilogue, (hipStream_t)stream);
}
