// Rotary positions: pairs of a head's elements turned by an angle that grows with the position, and the store of new
// tokens' keys (turned) and values into a decode cache.
//
// Pair i of a row at position t, elements (a, b), becomes amp * (a cos - b sin, a sin + b cos) with the angle t * w_i; the
// elements past the turned part of a head stay as they are.  Pairs are elements i and i + rot/2 (half) or 2i and 2i + 1
// (interleaved).  The gradient is the turn back, by -angle with the same amp.
//
// Angles: t reaches 10^6, so t * w_i in 32 bits would be off by up to 0.06; w_i comes as turns (w_i / 2 pi) in 64 bits,
// the product is taken modulo one turn in 64 bits, and only the rest, at most half a turn, goes to a 32-bit sine and
// cosine.  For float32 rows those are the library's (off by at most 2^-24.2 over 2^24 arguments of that range); 16-bit rows
// take the hardware's sine, off by 2^-22.9 there, half a step of their results being 2^-11 and 2^-8 of them.
//
// Bound by bytes: each element is read and written once.  A thread takes one unit of one row, two pieces of 16 bytes that lie
// half the turned part apart (single elements where rows are not whole such pieces), so that the threads of a row read and
// write whole runs of it.  The sines again for every head cost nothing beside the bytes: four heads of a token a thread, which
// share them, took 113 and 130 us for the sizes below, eight 116 and 144.  Stores are ordinary ones: what is written is read
// next.
//
// 30001 positions of 20 heads of 128 in float32, 614 MB: 106 us, 5.8 TB/s.  Prompts of 8 x 8191 tokens, 12 heads of 64, into
// pages of 64 rows in bfloat16 (queries turned too), 604 MB: 119 us, 5.1 TB/s.  One token of 32 sequences: 4.2 us, a launch.
// Turned parts that are not whole pieces go element by element: 8 x 24 heads of 64 x 8191 in bfloat16 209 us with 20 or 24
// elements turned, 1.9 TB/s, and 83 with all of them.
//
// The reference has learned positions only (model.py:54, 74); it stores keys and values at engine.py:41-55.
#include "common.hpp"

namespace ta {
namespace {

constexpr int kThreads = 256;

struct RowsOf {
  const void* p;
  int64_t sb, sh, st;
};

struct Rope {
  int rot;              // turned elements of a head, even
  const double* turns;  // (rot / 2) turns a position
  float amp;            // negative sine for the turn back
  float sign;
};

template <typename T> constexpr int vec_elems() { return 16 / (int)sizeof(T); }

// cos and sin of pos * turns (a whole number of turns taken off in 64 bits), both times amp.
template <typename T>
__device__ __forceinline__ void turn_of(const Rope& r, int pair, int pos, float& c, float& s) {
  const double x = (double)pos * r.turns[pair];
  const float f = (float)(x - rint(x));   // in [-0.5, 0.5]
  float sn, cs;
  if constexpr (__is_same(T, float)) {
    sincospif(2.0f * f, &sn, &cs);
  } else {
    sn = __builtin_amdgcn_sinf(f);        // the hardware's argument is in turns
    cs = __builtin_amdgcn_cosf(f);
  }
  c = cs * r.amp;
  s = sn * (r.amp * r.sign);
}

// A unit of a row: NE elements at a and NE at b, as pairs (a[i], b[i]) (half) or (a[2i], a[2i + 1]) and b's (interleaved);
// NE = 16 bytes' worth with VEC, else one element.
template <typename T, bool VEC> struct Unit {
  static constexpr int NE = VEC ? vec_elems<T>() : 1;
  alignas(VEC ? 16 : sizeof(T)) T a[NE];
  alignas(VEC ? 16 : sizeof(T)) T b[NE];
};

template <typename T, bool VEC>
__device__ __forceinline__ void unit_load(const T* row, int ia, int ib, Unit<T, VEC>& u) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(u.a) = ldg16(row + ia);
    *reinterpret_cast<uint4*>(u.b) = ldg16(row + ib);
  } else {
    u.a[0] = row[ia];
    u.b[0] = row[ib];
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void unit_store(T* row, int ia, int ib, const Unit<T, VEC>& u) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(row + ia) = *reinterpret_cast<const uint4*>(u.a);
    *reinterpret_cast<uint4*>(row + ib) = *reinterpret_cast<const uint4*>(u.b);
  } else {
    row[ia] = u.a[0];
    row[ib] = u.b[0];
  }
}
// One pair; the multiply-adds are written out, so that every form of the kernels gives the same bits.
template <typename T>
__device__ __forceinline__ void turn_pair(T& x, T& y, float c, float s) {
  const float a = to_f32(x), b = to_f32(y);
  x = from_f32<T>(fmaf(a, c, -(b * s)));
  y = from_f32<T>(fmaf(a, s, b * c));
}
// Unit u, turned: its pairs' angles from the position.
template <typename T, bool VEC, bool INTER>
__device__ __forceinline__ void unit_turn(Unit<T, VEC>& e, const Rope& r, int u, int pos) {
  constexpr int NE = Unit<T, VEC>::NE;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    float c, s;
    if constexpr (INTER && VEC) {
      const bool second = i >= NE / 2;
      const int k = i % (NE / 2);
      turn_of<T>(r, (second ? r.rot / 4 : 0) + u * (NE / 2) + k, pos, c, s);
      T* x = second ? e.b : e.a;
      turn_pair<T>(x[2 * k], x[2 * k + 1], c, s);
    } else {
      turn_of<T>(r, u * NE + i, pos, c, s);
      turn_pair<T>(e.a[i], e.b[i], c, s);
    }
  }
}

// Units of a row: the turned ones, then what is left of the head, two pieces a unit (the last may hold one).
template <typename T, bool VEC, bool INTER>
struct RowUnits {
  static constexpr int NE = Unit<T, VEC>::NE;
  int ia, ib;
  bool turn;
  __device__ __forceinline__ RowUnits(int u, int rot, int D) {
    const int turned = rot / (2 * NE);
    turn = u < turned;
    if (turn) {
      ia = INTER && !VEC ? 2 * u : u * NE;
      ib = INTER && !VEC ? ia + 1 : ia + rot / 2;
    } else {
      const int units = ((D - rot) / NE + 1) / 2;
      ia = rot + (u - turned) * NE;
      ib = ia + units * NE;
      if (ib >= D) ib = ia;
    }
  }
};
inline int row_units(int NE, int rot, int D) { return rot / (2 * NE) + ((D - rot) / NE + 1) / 2; }

struct RopeArgs {
  RowsOf x;
  void* y;
  int64_t ysb, ysh, yst;
  int H, T, D, units;
  int64_t n;            // units in all
  Rope r;
  const int32_t* pos;
  int64_t pos_sb;
};

template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs p) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.n) return;
  const int u = (int)(at % p.units);
  const int64_t rest = at / p.units;
  const int h = (int)(rest % p.H);
  const int64_t tok = rest / p.H;
  const int t = (int)(tok % p.T);
  const int64_t b = tok / p.T;
  const RowUnits<T, VEC, INTER> w(u, p.r.rot, p.D);
  Unit<T, VEC> e;
  unit_load<T, VEC>(reinterpret_cast<const T*>(p.x.p) + b * p.x.sb + h * p.x.sh + t * p.x.st, w.ia, w.ib, e);
  if (w.turn) unit_turn<T, VEC, INTER>(e, p.r, u, p.pos[b * p.pos_sb + t]);
  unit_store<T, VEC>(reinterpret_cast<T*>(p.y) + b * p.ysb + h * p.ysh + t * p.yst, w.ia, w.ib, e);
}

struct StoreArgs {
  RowsOf q, k, v;
  void* qo;
  int64_t osb, osh, ost;
  void* Kc;
  void* Vc;
  int64_t csb, csh, cst;
  const int32_t* ptab;
  int64_t pt_sb, pt_sh, pstride, npages;
  int blog2;
  int Hq, H, N, D, Tcap, units;
  int64_t n;
  Rope r;
  const int32_t* pos;
  int64_t pos_sb;
};

// As rope_kernel over the Hq query heads, the H key heads and the H value heads of a token; keys and values go to the row
// of the token's position in the cache (nowhere when it is outside the cache or its block has no page).
template <typename T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(StoreArgs p) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.n) return;
  const int u = (int)(at % p.units);
  const int64_t rest = at / p.units;
  const int heads = p.Hq + 2 * p.H, h = (int)(rest % heads);
  const int64_t tok = rest / heads;
  const int t = (int)(tok % p.N);
  const int64_t b = tok / p.N;
  const RowUnits<T, VEC, INTER> w(u, p.r.rot, p.D);
  const int pos = p.pos[b * p.pos_sb + t];
  const bool query = h < p.Hq, value = h >= p.Hq + p.H;
  const int hh = query ? h : h - p.Hq - (value ? p.H : 0);
  const RowsOf& src = query ? p.q : value ? p.v : p.k;
  Unit<T, VEC> e;
  unit_load<T, VEC>(reinterpret_cast<const T*>(src.p) + b * src.sb + hh * src.sh + t * src.st, w.ia, w.ib, e);
  T* to;
  if (query) {
    to = reinterpret_cast<T*>(p.qo) + b * p.osb + hh * p.osh + t * p.ost;
  } else {
    if (pos < 0 || pos >= p.Tcap) return;
    to = reinterpret_cast<T*>(value ? p.Vc : p.Kc);
    if (p.ptab == nullptr) {
      to += b * p.csb + hh * p.csh + pos * p.cst;
    } else {
      const int pg = p.ptab[b * p.pt_sb + hh * p.pt_sh + (pos >> p.blog2)];
      if (pg < 0 || pg >= p.npages) return;
      to += pg * p.pstride + (pos & ((1 << p.blog2) - 1)) * p.cst;
    }
  }
  if (w.turn && !value) unit_turn<T, VEC, INTER>(e, p.r, u, pos);
  unit_store<T, VEC>(to, w.ia, w.ib, e);
}

bool pieces(int sz, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return false;
  for (int64_t s : strides)
    if ((s * sz) % 16) return false;
  return true;
}

int check_rope(const char* who, int dtype, int D, int rot, const double* turns, const int32_t* pos) {
  if (dtype != TA_F32 && dtype != TA_F16 && dtype != TA_BF16) {
    set_error(std::string(who) + ": unknown dtype");
    return TA_ERR_ARG;
  }
  if (D < 1 || D > 65536 || rot < 0 || rot > D || rot % 2 || (rot > 0 && (turns == nullptr || (uintptr_t)turns % 8)) ||
      pos == nullptr) {
    set_error(std::string(who) + ": bad sizes (an even number of turned elements, at most the head) or a missing pointer");
    return TA_ERR_ARG;
  }
  return TA_OK;
}

// Workgroups for `n` units; 0 (and the error set): too many.
unsigned grid_of(const char* who, int64_t n) {
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) {
    set_error(std::string(who) + ": too large");
    return 0;
  }
  return (unsigned)blocks;
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_rope(const void* x, int dtype, int64_t xsb, int64_t xsh, int64_t xst, void* y, int64_t ysb, int64_t ysh,
                       int64_t yst, int B, int H, int T, int D, int rot, const double* turns, int interleaved, float amp,
                       int inverse, const int32_t* pos, int64_t pos_sb, void* stream) {
  const int rc = check_rope("ta_rope", dtype, D, rot, turns, pos);
  if (rc != TA_OK) return rc;
  if (B < 0 || H < 0 || T < 0 || x == nullptr || y == nullptr) {
    set_error("ta_rope: bad sizes or a missing pointer");
    return TA_ERR_ARG;
  }
  if (B == 0 || H == 0 || T == 0) return TA_OK;
  const int sz = dtype == TA_F32 ? 4 : 2;
  const int ne = 16 / sz;
  const bool vec = rot % (2 * ne) == 0 && D % ne == 0 && pieces(sz, {x, y}, {xsb, xsh, xst, ysb, ysh, yst});
  RopeArgs p{{x, xsb, xsh, xst}, y, ysb, ysh, yst, H, T, D, row_units(vec ? ne : 1, rot, D), 0,
             {rot, turns, amp, inverse ? -1.0f : 1.0f}, pos, pos_sb};
  p.n = (int64_t)B * T * H * p.units;
  const unsigned blocks = grid_of("ta_rope", p.n);
  if (!blocks) return TA_ERR_UNSUPPORTED;
#define TA_ROPE(TT, V, I) \
  hipLaunchKernelGGL((rope_kernel<TT, V, I>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p)
#define TA_ROPE_T(TT)                                          \
  do {                                                         \
    if (vec && interleaved) TA_ROPE(TT, true, true);           \
    else if (vec) TA_ROPE(TT, true, false);                    \
    else if (interleaved) TA_ROPE(TT, false, true);            \
    else TA_ROPE(TT, false, false);                            \
  } while (0)
  switch (dtype) {
    case TA_F32: TA_ROPE_T(float); break;
    case TA_F16: TA_ROPE_T(f16_t); break;
    default: TA_ROPE_T(bf16_t); break;
  }
#undef TA_ROPE
#undef TA_ROPE_T
  return check_launch("rope_kernel");
}

extern "C" int ta_kv_store(const void* k, const void* v, int dtype, int64_t ksb, int64_t ksh, int64_t kst, int64_t vsb,
                           int64_t vsh, int64_t vst, const void* q, int64_t qsb, int64_t qsh, int64_t qst, void* q_out,
                           int64_t osb, int64_t osh, int64_t ost, int Hq, void* Kc, void* Vc, int64_t csb, int64_t csh,
                           int64_t cst, int B, int H, int N, int D, int Tcap, const int32_t* pos, int64_t pos_sb, int rot,
                           const double* turns, int interleaved, float amp, const ta_kv_pages* pages, void* stream) {
  const int rc = check_rope("ta_kv_store", dtype, D, rot, turns, pos);
  if (rc != TA_OK) return rc;
  if (B < 0 || H < 1 || N < 0 || Hq < 0 || Tcap < 1 || k == nullptr || v == nullptr || Kc == nullptr || Vc == nullptr ||
      (Hq > 0 && (q == nullptr || q_out == nullptr)) || Hq > (1 << 28) || H > (1 << 28)) {
    set_error("ta_kv_store: bad sizes or a missing pointer");
    return TA_ERR_ARG;
  }
  if (pages && (pages->table == nullptr || pages->num_pages <= 0 || pages->block_log2 < 0 || pages->block_log2 > 14 ||
                pages->page_stride < (cst << pages->block_log2))) {
    set_error("ta_kv_store: bad page description");
    return TA_ERR_ARG;
  }
  if (B == 0 || N == 0) return TA_OK;
  const int sz = dtype == TA_F32 ? 4 : 2;
  const int ne = 16 / sz;
  bool vec = rot % (2 * ne) == 0 && D % ne == 0 && pieces(sz, {k, v, Kc, Vc}, {ksb, ksh, kst, vsb, vsh, vst, cst}) &&
             (Hq == 0 || pieces(sz, {q, q_out}, {qsb, qsh, qst, osb, osh, ost})) &&
             (pages ? pieces(sz, {}, {pages->page_stride}) : pieces(sz, {}, {csb, csh}));
  StoreArgs p{{q, qsb, qsh, qst}, {k, ksb, ksh, kst}, {v, vsb, vsh, vst}, q_out, osb, osh, ost, Kc, Vc, csb, csh, cst,
              nullptr, 0, 0, 0, 0, 0, Hq, H, N, D, Tcap, row_units(vec ? ne : 1, rot, D), 0,
              {rot, turns, amp, 1.0f}, pos, pos_sb};
  if (pages) {
    p.ptab = pages->table;
    p.pt_sb = pages->sb;
    p.pt_sh = pages->sh;
    p.pstride = pages->page_stride;
    p.npages = pages->num_pages;
    p.blog2 = pages->block_log2;
  }
  p.n = (int64_t)B * N * (Hq + 2 * H) * p.units;
  const unsigned blocks = grid_of("ta_kv_store", p.n);
  if (!blocks) return TA_ERR_UNSUPPORTED;
#define TA_STORE(TT, V, I) \
  hipLaunchKernelGGL((kv_store_kernel<TT, V, I>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p)
#define TA_STORE_T(TT)                                         \
  do {                                                         \
    if (vec && interleaved) TA_STORE(TT, true, true);          \
    else if (vec) TA_STORE(TT, true, false);                   \
    else if (interleaved) TA_STORE(TT, false, true);           \
    else TA_STORE(TT, false, false);                           \
  } while (0)
  switch (dtype) {
    case TA_F32: TA_STORE_T(float); break;
    case TA_F16: TA_STORE_T(f16_t); break;
    default: TA_STORE_T(bf16_t); break;
  }
#undef TA_STORE
#undef TA_STORE_T
  return check_launch("kv_store_kernel");
}
