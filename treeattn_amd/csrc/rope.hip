// Rotary positions: pairs of a head's elements turned by an angle that grows with the position, and the store of new
// tokens' keys (turned) and values into a decode cache.
//
// Pair i of a row at position t, elements (a, b), becomes amp * (a cos - b sin, a sin + b cos) with the angle t * w_i; the
// elements past the turned part of a head stay as they are.  Pairs are elements i and i + rot/2 (half) or 2i and 2i + 1
// (interleaved).  The gradient is the turn back, by -angle with the same amp.
//
// Angles: t reaches 10^6, so t * w_i in 32 bits would be off by up to 0.06; w_i comes as turns (w_i / 2 pi) in 64 bits,
// the product is taken modulo one turn in 64 bits, and only the rest, at most half a turn, goes to a 32-bit sine and
// cosine.  For float32 rows those are the library's (2^-23 of it); 16-bit rows take the hardware's sine, whose error
// (measured 2^-21 absolute) is far below half a step of the result (2^-12 and 2^-9 of it).
//
// Bound by bytes: each element is read and written once.  A thread holds one unit, 16 bytes of each half of some pairs
// (single elements where rows are not whole 16-byte pieces), and takes it through several heads of its token, which share
// its sines: with one head a thread the sines cost more than the bytes.
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

// A unit of a row: NE elements at a and NE at b, as pairs (a[i], b[i]) (half) or (a[2i], a[2i + 1]), then b's (interleaved);
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
template <typename T, bool VEC, bool INTER>
__device__ __forceinline__ void unit_turn(Unit<T, VEC>& u, const float* c, const float* s) {
  constexpr int NE = Unit<T, VEC>::NE;
  if constexpr (INTER && VEC) {
#pragma unroll
    for (int i = 0; i < NE / 2; ++i) {
      turn_pair<T>(u.a[2 * i], u.a[2 * i + 1], c[i], s[i]);
      turn_pair<T>(u.b[2 * i], u.b[2 * i + 1], c[NE / 2 + i], s[NE / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NE; ++i) turn_pair<T>(u.a[i], u.b[i], c[i], s[i]);
  }
}

// Units of a row: the turned ones, then what is left of the head, two pieces a unit (the last may hold one).
template <typename T, bool VEC, bool INTER>
struct RowUnits {
  static constexpr int NE = Unit<T, VEC>::NE;
  int turned, rest, ia, ib;   // rest: pieces past the turned part
  bool turn, two;
  __device__ __forceinline__ RowUnits(int u, int rot, int D) {
    turned = rot / (2 * NE);
    turn = u < turned;
    two = true;
    if (turn) {
      ia = INTER ? u * 2 * NE : u * NE;
      ib = INTER ? ia + NE : ia + rot / 2;
    } else {
      ia = rot + (u - turned) * 2 * NE;
      ib = ia + NE;
      two = ib < D;
      if (!two) ib = ia;
    }
  }
};
inline int row_units(int NE, int rot, int D) { return rot / (2 * NE) + ((D - rot) / NE + 1) / 2; }

struct RopeArgs {
  RowsOf x;
  void* y;
  int64_t ysb, ysh, yst;
  int H, T, D, units, groups;   // groups of heads a token
  int64_t n;                    // threads' worth of work
  Rope r;
  const int32_t* pos;
  int64_t pos_sb;
};

// HPT heads of one token a thread, the same unit of each.
template <typename T, bool VEC, bool INTER, int HPT>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs p) {
  using U = Unit<T, VEC>;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.n) return;
  const int u = (int)(at % p.units);
  const int64_t rest = at / p.units;
  const int g = (int)(rest % p.groups);
  const int64_t tok = rest / p.groups;
  const int t = (int)(tok % p.T);
  const int64_t b = tok / p.T;
  const RowUnits<T, VEC, INTER> w(u, p.r.rot, p.D);
  const T* x = reinterpret_cast<const T*>(p.x.p) + b * p.x.sb + t * p.x.st;
  T* y = reinterpret_cast<T*>(p.y) + b * p.ysb + t * p.yst;
  U e[HPT];
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = g + j * p.groups;
    if (h < p.H) unit_load<T, VEC>(x + h * p.x.sh, w.ia, w.ib, e[j]);
  }
  if (w.turn) {
    float c[U::NE], s[U::NE];
    const int pos = p.pos[b * p.pos_sb + t];
#pragma unroll
    for (int i = 0; i < U::NE; ++i) turn_of<T>(p.r, u * U::NE + i, pos, c[i], s[i]);
#pragma unroll
    for (int j = 0; j < HPT; ++j) unit_turn<T, VEC, INTER>(e[j], c, s);
  }
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = g + j * p.groups;
    if (h < p.H) unit_store<T, VEC>(y + h * p.ysh, w.ia, w.ib, e[j]);
  }
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
  int Hq, H, N, D, Tcap, units, groups;
  int64_t n;
  Rope r;
  const int32_t* pos;
  int64_t pos_sb;
};

// As rope_kernel over the Hq query heads, the H key heads and the H value heads of a token; keys and values go to the row
// of the token's position in the cache (nowhere when it is outside the cache or its block has no page).
template <typename T, bool VEC, bool INTER, int HPT>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(StoreArgs p) {
  using U = Unit<T, VEC>;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.n) return;
  const int u = (int)(at % p.units);
  const int64_t rest = at / p.units;
  const int g = (int)(rest % p.groups);
  const int64_t tok = rest / p.groups;
  const int t = (int)(tok % p.N);
  const int64_t b = tok / p.N;
  const RowUnits<T, VEC, INTER> w(u, p.r.rot, p.D);
  const int pos = p.pos[b * p.pos_sb + t];
  const bool in = pos >= 0 && pos < p.Tcap;
  const int heads = p.Hq + 2 * p.H;
  U e[HPT];
  int64_t to[HPT];     // the row's place in the cache, -1: none
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = g + j * p.groups;
    to[j] = -1;
    if (h >= heads) continue;
    const RowsOf& src = h < p.Hq ? p.q : (h < p.Hq + p.H ? p.k : p.v);
    const int hh = h < p.Hq ? h : (h - p.Hq) % p.H;
    unit_load<T, VEC>(reinterpret_cast<const T*>(src.p) + b * src.sb + hh * src.sh + t * src.st, w.ia, w.ib, e[j]);
    if (h >= p.Hq && in) {
      if (p.ptab == nullptr) {
        to[j] = b * p.csb + hh * p.csh + pos * p.cst;
      } else {
        const int pg = p.ptab[b * p.pt_sb + hh * p.pt_sh + (pos >> p.blog2)];
        if (pg >= 0 && pg < p.npages) to[j] = pg * p.pstride + (pos & ((1 << p.blog2) - 1)) * p.cst;
      }
    }
  }
  if (w.turn) {
    float c[U::NE], s[U::NE];
#pragma unroll
    for (int i = 0; i < U::NE; ++i) turn_of<T>(p.r, u * U::NE + i, pos, c[i], s[i]);
#pragma unroll
    for (int j = 0; j < HPT; ++j)
      if (g + j * p.groups < p.Hq + p.H) unit_turn<T, VEC, INTER>(e[j], c, s);
  }
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = g + j * p.groups;
    if (h < p.Hq)
      unit_store<T, VEC>(reinterpret_cast<T*>(p.qo) + b * p.osb + h * p.osh + t * p.ost, w.ia, w.ib, e[j]);
    else if (to[j] >= 0)
      unit_store<T, VEC>(reinterpret_cast<T*>(h < p.Hq + p.H ? p.Kc : p.Vc) + to[j], w.ia, w.ib, e[j]);
  }
}

// Heads a thread: four where that leaves enough threads for the whole GPU, else one (the sines again for every head).
constexpr int kHeads = 4;
constexpr int64_t kEnough = (int64_t)1 << 19;

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

template <typename F>
int grid_of(const char* who, int64_t tokens, int heads, int units, int& groups, int64_t& n, bool& many, F f) {
  const int64_t one = tokens * heads;
  many = one * units >= kEnough * kHeads;
  groups = many ? (heads + kHeads - 1) / kHeads : heads;
  n = tokens * groups * units;
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) {
    set_error(std::string(who) + ": too large");
    return TA_ERR_UNSUPPORTED;
  }
  f((unsigned)blocks);
  return check_launch(who);
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
  RopeArgs p{{x, xsb, xsh, xst}, y, ysb, ysh, yst, H, T, D, row_units(vec ? ne : 1, rot, D), 0, 0,
             {rot, turns, amp, inverse ? -1.0f : 1.0f}, pos, pos_sb};
  bool many;
  return grid_of("ta_rope", (int64_t)B * T, H, p.units, p.groups, p.n, many, [&](unsigned blocks) {
#define TA_ROPE(TT, V, I)                                                                                              \
  do {                                                                                                                 \
    if (many) hipLaunchKernelGGL((rope_kernel<TT, V, I, kHeads>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p); \
    else hipLaunchKernelGGL((rope_kernel<TT, V, I, 1>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p);       \
  } while (0)
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
  });
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
              nullptr, 0, 0, 0, 0, 0, Hq, H, N, D, Tcap, row_units(vec ? ne : 1, rot, D), 0, 0,
              {rot, turns, amp, 1.0f}, pos, pos_sb};
  if (pages) {
    p.ptab = pages->table;
    p.pt_sb = pages->sb;
    p.pt_sh = pages->sh;
    p.pstride = pages->page_stride;
    p.npages = pages->num_pages;
    p.blog2 = pages->block_log2;
  }
  bool many;
  return grid_of("ta_kv_store", (int64_t)B * N, Hq + 2 * H, p.units, p.groups, p.n, many, [&](unsigned blocks) {
#define TA_STORE(TT, V, I)                                                                                          \
  do {                                                                                                              \
    if (many)                                                                                                       \
      hipLaunchKernelGGL((kv_store_kernel<TT, V, I, kHeads>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p); \
    else                                                                                                            \
      hipLaunchKernelGGL((kv_store_kernel<TT, V, I, 1>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream, p);  \
  } while (0)
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
  });
}
