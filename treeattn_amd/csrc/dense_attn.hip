// Attention of new tokens over a whole decode cache: every key from position 0 to the query's own.
//
//   s_j = scale * (q . k_j),  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse = m + log sum_j e^(s_j - m)
//
// over the keys j = 0 .. t that have a page.  Query head h reads key head h / (Hq / H).  Scores, sums and the accumulators
// are float32, the output is rounded once.
//
// One pass over the keys with a running maximum and sum, on the matrix cores even for a single query: the 16 rows of a tile
// are the query heads of a key head times the new tokens, and what a lone row wastes of the instructions is less than the
// vector units would take (32 keys of 64: 12 instructions of 16 cycles, against some 150 of 4).  Scores and weights
// stay in registers: with S^T = K Q^T a lane holds four scores of one query row, which are what the next product, O^T = V^T P^T, takes as
// its B operand when that product counts the keys in the order the first leaves them in; V^T's operand is a lane's eight
// keys at its own columns, turned round in registers; the running maximum, the sum and their corrections are then one
// number a lane.
//
// Weights of 16-bit rows go into the second product as the sum of two 16-bit numbers (2^-17 of a weight is lost, where
// one would lose 2^-9, as much as the rounding of the result).  The maximum is renewed only when a score passes it by more
// than kSlack: until then weights are at most 2^kSlack.
//
// Bound by bytes, 2 D a key and key head, where rows are few; the keys of a sequence are split over wavefronts and
// workgroups, whose partial results the last workgroup to arrive joins.  32 x 12 queries over 32768 keys of 64: 441 us, 6.4
// TB/s; one sequence of 131000: 59 us, 5.9 TB/s.  Rows of prompts, by the hundred, share their keys through LDS (Block).
// (Times beside a choice are of one session, both sides; the same call differs by up to 10 % between sessions.)
//
// Phase marks (trace.hpp): 0 start, 1 its part and queries are known, 2 its keys are done, 3 its part is written, 4 it is
// counted in, 5 the set is joined.
//
// Reference functions replaced: engine.py:74-81 (DenseState.attend).
#include "attn.hpp"
#include "trace.hpp"

namespace ta {
namespace {

constexpr float kLowest = -3.4028235e38f;

struct Dense {
  const void* q;
  int64_t qsb, qsh, qsn;
  const void* k;
  int64_t ksb, ksh, kst;
  const void* v;
  int64_t vsb, vsh, vst;
  int Hq, H, G, Nq, D, Tk;
  const int32_t* tq;
  int64_t tq_sb;
  float scale;
  void* out;
  int64_t osb, osh, osn;
  float* lse;
  // pages (ptab != null): block j of (b, h) is page ptab[b * pt_sb + h * pt_sh + j], its row r at k + page * pstride + r * kst
  const int32_t* ptab;
  int64_t pt_sb, pt_sh, pstride, npages;
  int blog2;
  int BH, R;            // (sequence, key head) pairs; query rows of one: G * Nq
  int B;
  float* ws;            // parts (workgroup, row, D + 2) and
  uint32_t* cnt;        // arrival counters of the sets (zero between calls)
  int2* heads;          // of many rows' sets: the first part, and how many
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kRows = 16;            // query rows of a tile
constexpr float kLittle = -24.0f;    // log2 of the largest weight where sums would pass the range of a float
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T, int D, bool MANY = false> struct Tile {
  static constexpr int EB = (int)sizeof(T);
  // Tiles of 16 keys a step.  Heads of 128 take one: two steps of 32 keys in registers leave no room for two wavefronts on a
  // SIMD (256 registers and spills).  MANY: the steps stand in LDS.
  static constexpr int KT = MANY ? 4 : D == 128 ? 1 : 2;
  static constexpr int KEYS = 16 * KT;
  static constexpr int KS = EB == 2 ? (D + 31) / 32 : D / 16;   // 16-byte pieces of a key row a lane
  static constexpr int DJ = D / 16;                             // columns of V a lane holds
  static constexpr int VB = DJ * EB;                            // their bytes, of one key
  static constexpr int VW = (VB + 3) / 4;
  // LDS bytes of a key row (16 more than the row, so that 8 rows' pieces lie in different banks) and of a wavefront's step
  static constexpr int LROW = (D * EB < 64 ? 64 : D * EB) + 16;
  static constexpr int LSTEP = KEYS * LROW;
  // weights are exp2(x - max + kShift): float16 keeps 2^-24 absolutely, which is far below the largest weight then
  static constexpr float kShift = __is_same(T, f16_t) ? 10.0f : 0.0f;
  static constexpr float kSlack = __is_same(T, f16_t) ? 4.0f : 8.0f;
};

// The keys and values of one step, in a lane: K rows 16 i + lane / 4 at pieces lane % 4 (four lanes next to each other read 64
// bytes of a row); V rows 16 i + 4 (lane / 16) + u at columns DJ (lane % 16) ...
template <typename T, int D, bool MANY = false> struct Step {
  using C = Tile<T, D, MANY>;
  uint4 k[C::KT][C::KS];
  uint32_t v[MANY ? 1 : C::KT * 4][C::VW];
  uint32_t have;     // bit 4 i + u: key 16 i + 4 (lane / 16) + u has a page
  int key0;
};

template <typename T>
__device__ __forceinline__ f32x4 mfma32(const uint4& a, const uint4& b, f32x4 c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x2 a, u32x2 b, f32x4 c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

// two floats rounded to two elements of T, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, f16_t)) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
  } else {
    return bf16_pack2(a, b);
  }
}
template <typename T>
__device__ __forceinline__ float unpack_lo(uint32_t x) {
  if constexpr (__is_same(T, f16_t)) return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
  else return __uint_as_float(x << 16);
}
template <typename T>
__device__ __forceinline__ float unpack_hi(uint32_t x) {
  if constexpr (__is_same(T, f16_t)) return (float)__builtin_bit_cast(_Float16, (uint16_t)(x >> 16));
  else return __uint_as_float(x & 0xffff0000u);
}

// What is left of two weights once their two halves of hi are taken off.
template <typename T>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t hi) {
  if constexpr (__is_same(T, f16_t)) {
    return pack2<T>(a - unpack_lo<T>(hi), b - unpack_hi<T>(hi));
  } else {
    // a - 1 x one half - 0 x the other, exact (weights are finite); the factors from registers, since as an inline constant the
    // compiler's -1 of the lower half is the instruction's of the upper one
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 h = __builtin_bit_cast(bf16x2, hi);
    uint32_t first = 0x0000bf80u, second = 0xbf800000u;
    asm("" : "+s"(first), "+s"(second));
    return pack2<T>(__builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), a, false),
                    __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), b, false));
  }
}

// The larger / the sum of x over the four lanes that share lane % 16.
__device__ __forceinline__ float max_rows(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_rows(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a pass over the keys takes for values: what is there; with a weight of 1 for every key that a row sees, ones where it is
// infinite with the sign or NaN and zeros elsewhere (kUp, kDown); zeros where it is infinite or NaN (kFinite, and kSmall, whose
// weights are at most 2^-24).
enum Values { kAll, kUp, kDown, kFinite, kSmall };

// Those values in place of x's two 16-bit ones (one of 32 bits).
template <typename T>
__device__ __forceinline__ uint32_t stand_in(uint32_t x, Values values) {
  constexpr bool wide = sizeof(T) == 4;
  constexpr uint32_t kExp = wide ? 0x7f800000u : __is_same(T, f16_t) ? 0x7c00u : 0x7f80u;
  constexpr uint32_t kOne = wide ? 0x3f800000u : __is_same(T, f16_t) ? 0x3c00u : 0x3f80u;
  constexpr uint32_t kAbs = wide ? 0x7fffffffu : 0x7fffu;
  auto one = [&](uint32_t h) {
    const bool not_finite = (h & kExp) == kExp;
    if (values >= kFinite) return not_finite ? 0u : h;
    const bool sign = values == kUp ? h <= kAbs : h > kAbs;
    return not_finite && (sign || (h & kAbs) != kExp) ? kOne : 0u;
  };
  if constexpr (wide) return one(x);
  else return one(x & 0xffffu) | one(x >> 16) << 16;
}

// Row r of a key head's query rows: query head j of its group, token n.
__device__ __forceinline__ void head_token(const Dense& p, int r, int& j, int& n) {
  j = p.Nq == 1 ? r : r / p.Nq;
  n = p.Nq == 1 ? 0 : r - j * p.Nq;
}

// The smaller of x over 16 lanes.
template <int CTRL>
__device__ __forceinline__ int min_dpp(int x) {
  const int y = __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false);
  return y < x ? y : x;
}
__device__ __forceinline__ int min16(int x) { return min_dpp<0x140>(min_dpp<0x141>(min_dpp<0x4E>(min_dpp<0xB1>(x)))); }

// A load that the caches need not keep (STREAM), or an ordinary one.
template <bool STREAM, typename V>
__device__ __forceinline__ V once(const TA_GLOBAL V* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

// One wavefront's share: keys [k0, k1) for NT tiles of 16 query rows of one (sequence, key head).
template <typename T, int D, bool WIDE, int NT, bool MANY = false>
struct Share {
  using C = Tile<T, D, MANY>;
  const Dense& p;
  const int lane, c, g;
  const TA_GLOBAL T* kb;
  const TA_GLOBAL T* vb;
  const int32_t* tab;
  int t[NT];            // the lane's row's position; of rows that are not there or see nothing: behind every key
  uint32_t none;        // rows (bit 16 i + c) whose position is outside the cache: zeros
  int tmin, tmax;       // of the wavefront's rows; values past the last count as zeros
  uint4 q[NT][C::KS];
  f32x4 acc[NT][C::DJ];
  float m[NT], l[NT];   // the reference of the weights (max - kShift), and the lane's part of their sum
  char* lds;            // this wavefront's LSTEP bytes
  int pg;               // page (WIDE), or the page of key lane % 32, of the step that is fetched next

  __device__ __forceinline__ Share(const Dense& p_, int b, int h, int row0, char* lds_, bool one = false, int last = -1)
      : p(p_), lane(lane_id()), c(lane & 15), g(lane >> 4), lds(lds_) {
    kb = (const TA_GLOBAL T*)p.k + (p.ptab ? 0 : b * p.ksb + h * p.ksh);
    vb = (const TA_GLOBAL T*)p.v + (p.ptab ? 0 : b * p.vsb + h * p.vsh);
    tab = p.ptab ? p.ptab + b * p.pt_sb + h * p.pt_sh : nullptr;
    int lo = 0x7fffffff, hi = -1;
    none = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = row0 + kRows * i + c;
      const bool in = r < p.R;
      int j = 0, n = 0;
      if (in) head_token(p, r, j, n);
      int tt = 0x7fffffff;
      if (in) {
        tt = one ? last : p.tq[b * p.tq_sb + n];   // (one token: its position, checked, is known)
      }
      // (masks would be needed for such a row's sake in every step: it goes along with the others instead)
      const bool out = in && (tt < 0 || tt >= p.Tk);
      none |= (uint32_t)(__ballot(out) & 0xffff) << (kRows * i);
      if (out) tt = 0x7fffffff;
      t[i] = tt;
      lo = tt < lo ? tt : lo;
      hi = tt != 0x7fffffff && tt > hi ? tt : hi;
      const T* qr = reinterpret_cast<const T*>(p.q) + b * p.qsb + (int64_t)(h * p.G + j) * p.qsh + n * p.qsn;
#pragma unroll
      for (int s = 0; s < C::KS; ++s) {
        const int d = C::EB == 2 ? 32 * s + 8 * g : 16 * s + 4 * g;
        q[i][s] = in && d < D ? ldg16(qr + d) : make_uint4(0, 0, 0, 0);
        if (p.scale < 0.0f) {
          const uint32_t sign = C::EB == 2 ? 0x80008000u : 0x80000000u;
          q[i][s].x ^= sign;
          q[i][s].y ^= sign;
          q[i][s].z ^= sign;
          q[i][s].w ^= sign;
        }
      }
    }
    reset();
    lo = min16(lo);
    hi = -min16(-hi);
    tmin = __builtin_amdgcn_readfirstlane(lo);
    tmax = __builtin_amdgcn_readfirstlane(hi);
  }

  __device__ __forceinline__ int page_of(int key0) const {
    if (WIDE) return tab ? tab[key0 >> p.blog2] : 0;
    const int key = key0 + (lane & 31);
    return tab[(key < tmax ? key : tmax) >> p.blog2];
  }

  // Requests step x's rows (keys key0 ...) from the pages in pg, and before them the pages of the step at next0.  A step that
  // is not needed (past the last one; loads are not left out, so that what is waited for is a fixed number of loads) reads one
  // row of its first key.
  template <bool STREAM>
  __device__ __forceinline__ void fetch(Step<T, D>& x, int key0, int next0, bool live) {
    x.key0 = key0;
    const int mine = pg;
    pg = page_of(next0);
    __builtin_amdgcn_sched_barrier(0);
    auto load_k = [&](int i, int s2, const TA_GLOBAL char* row) {
      const int o = 64 * s2 + 16 * (lane & 3);
      const u32x4_t r = once<STREAM>((const TA_GLOBAL u32x4_t*)(row + (uint32_t)(o < D * C::EB ? o : 0)));
      x.k[i][s2] = make_uint4(r.x, r.y, r.z, r.w);
    };
    auto load_v = [&](int e, const TA_GLOBAL char* at) {
      if constexpr (C::VB >= 16) {
#pragma unroll
        for (int w = 0; w < C::VW; w += 4) {
          const u32x4_t r = once<STREAM>((const TA_GLOBAL u32x4_t*)(at + 4 * w));
          x.v[e][w] = r.x;
          x.v[e][w + 1] = r.y;
          x.v[e][w + 2] = r.z;
          x.v[e][w + 3] = r.w;
        }
      } else if constexpr (C::VB == 8) {
        const u32x2 r = once<STREAM>((const TA_GLOBAL u32x2*)at);
        x.v[e][0] = r.x;
        x.v[e][1] = r.y;
      } else if constexpr (C::VB == 4) {
        x.v[e][0] = once<STREAM>((const TA_GLOBAL uint32_t*)at);
      } else {
        x.v[e][0] = once<STREAM>((const TA_GLOBAL uint16_t*)at);
      }
    };
    if constexpr (WIDE) {
      int64_t ko, vo;
      bool ok = true;
      // offsets of a step's rows in 32 bits, from one base; a contiguous cache may end inside a step: the last row that any
      // query sees in place of those behind it
      uint32_t klast = 0xffffffffu, vlast = 0xffffffffu;
      const uint32_t ks = (uint32_t)p.kst * C::EB, vs = (uint32_t)p.vst * C::EB;
      if (tab) {
        const int page = __builtin_amdgcn_readfirstlane(mine);
        ok = page >= 0 && page < p.npages;
        const int64_t to = (ok ? page : 0) * p.pstride;
        const int r = key0 & ((1 << p.blog2) - 1);
        ko = to + r * p.kst;
        vo = to + r * p.vst;
      } else {
        ko = key0 * p.kst;
        vo = key0 * p.vst;
        klast = (uint32_t)(tmax - key0) * ks;
        vlast = (uint32_t)(tmax - key0) * vs;
        if (tmax - key0 >= C::KEYS) klast = vlast = 0xffffffffu;
      }
      if (!live) klast = vlast = 0;
      x.have = ok ? 0xffffffffu : 0u;
      const TA_GLOBAL char* k0p = (const TA_GLOBAL char*)(kb + ko);
      const TA_GLOBAL char* v0p = (const TA_GLOBAL char*)(vb + vo);
#pragma unroll
      for (int i = 0; i < C::KT; ++i) {
        const uint32_t o = (lane >> 2) * ks + 16 * i * ks;
#pragma unroll
        for (int s2 = 0; s2 < C::KS; ++s2) load_k(i, s2, k0p + (o < klast ? o : klast));
      }
#pragma unroll
      for (int e = 0; e < C::KT * 4; ++e) {
        const uint32_t o = 4 * g * vs + (16 * (e / 4) + e % 4) * vs;
        load_v(e, v0p + ((o < vlast ? o : vlast) + C::VB * c));
      }
    } else {
      const int mask = live ? (1 << p.blog2) - 1 : 0;
      x.have = 0;
#pragma unroll
      for (int i = 0; i < C::KT; ++i) {
        int page = __shfl(mine, 16 * i + (lane >> 2), kWave);
        page = page >= 0 && page < p.npages && live ? page : 0;
        const TA_GLOBAL T* row = kb + page * p.pstride + (int64_t)((key0 + 16 * i + (lane >> 2)) & mask) * p.kst;
#pragma unroll
        for (int s2 = 0; s2 < C::KS; ++s2) load_k(i, s2, (const TA_GLOBAL char*)row);
      }
#pragma unroll
      for (int e = 0; e < C::KT * 4; e += 2) {
        const int key = 16 * (e / 4) + 4 * g + e % 4;
        const int page = __shfl(mine, key, kWave);
        const bool ok = page >= 0 && page < p.npages;
        x.have |= ok ? 3u << e : 0u;
        const TA_GLOBAL T* at = vb + (ok && live ? page : 0) * p.pstride;
        load_v(e, (const TA_GLOBAL char*)(at + (int64_t)((key0 + key) & mask) * p.vst) + C::VB * c);
        load_v(e + 1, (const TA_GLOBAL char*)(at + (int64_t)((key0 + key + 1) & mask) * p.vst) + C::VB * c);
      }
    }
  }

  // The step's keys from the lanes that loaded them to the lanes whose operand they are: lane (c, g) takes piece g of row c.
  // (Loaded in that order, each 16 bytes would be an access of their own to the first cache, which a piece of a prompt was
  // bound by: 371 accesses a step of 32 keys of 64 by a counter, now some 190.)
  __device__ __forceinline__ void turn(Step<T, D>& x) const {
    wave_sync();
#pragma unroll
    for (int a = 0; a < C::KT; ++a)
#pragma unroll
      for (int e = 0; e < C::KS; ++e)
        *reinterpret_cast<uint4*>(lds + (16 * a + (lane >> 2)) * C::LROW + 64 * e + 16 * (lane & 3)) = x.k[a][e];
    wave_sync();
#pragma unroll
    for (int a = 0; a < C::KT; ++a)
#pragma unroll
      for (int e = 0; e < C::KS; ++e)
        x.k[a][e] = *reinterpret_cast<const uint4*>(lds + (16 * a + c) * C::LROW + 64 * e + 16 * g);
  }

  // Scores of tile row set i: in lane (c, g) those of row c and keys 16 a + 4 g + u.
  __device__ __forceinline__ void scores(const Step<T, D, MANY>& x, int i, f32x4 (&s)[C::KT]) const {
#pragma unroll
    for (int a = 0; a < C::KT; ++a) {
      s[a] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < C::KS; ++e) {
        if constexpr (C::EB == 2) {
          uint4 k = x.k[a][e];
          if (D < 32 && g >= D / 8) k = make_uint4(0, 0, 0, 0);
          s[a] = mfma32<T>(k, q[i][e], s[a]);
        } else {
          const float* kf = reinterpret_cast<const float*>(&x.k[a][e]);
          const float* qf = reinterpret_cast<const float*>(&q[i][e]);
#pragma unroll
          for (int u = 0; u < 4; ++u) s[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[u], qf[u], s[a], 0, 0, 0);
        }
      }
    }
  }

  __device__ __forceinline__ bool sees(const Step<T, D, MANY>& x, int i, int a, int u) const {
    return x.key0 + 16 * a + 4 * g + u <= t[i] && (x.have >> (4 * a + u)) & 1;
  }

  // The weights of row set i in place of its scores (0 where masked), the running maximum renewed when one passes it by more
  // than kSlack.  AGAIN: for the values of `values`.
  template <bool MASKED, bool AGAIN>
  __device__ __forceinline__ void weights(const Step<T, D>& x, int i, f32x4 (&s)[C::KT], Values values) {
    if (AGAIN && values <= kDown) {
#pragma unroll
      for (int a = 0; a < C::KT; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[a][u] = sees(x, i, a, u) ? 1.0f : 0.0f;
      return;
    }
    const float shift = AGAIN && values == kSmall ? kLittle : C::kShift;
    const float past = AGAIN && values == kSmall ? kLittle : C::kShift + C::kSlack;
    const float f = fabsf(p.scale) * kLog2e;   // (a negative scale turns q round: the largest score is the largest product)
    float top = kLowest;
#pragma unroll
    for (int a = 0; a < C::KT; ++a)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (!MASKED || sees(x, i, a, u)) top = fmaxf(top, s[a][u]);
    top = top > kLowest ? top * f : kLowest;   // (a scale of zero, and products below the range, as others)
    if (__ballot(top > m[i] + past) != 0) {
      // only the rows that need it: what a row gives does not depend on the others
      const float mx = max_rows(top);
      const float mn = mx > m[i] + past ? mx - shift : m[i];
      const float alpha = __builtin_amdgcn_exp2f(m[i] - mn);
      m[i] = mn;
      l[i] *= alpha;
#pragma unroll
      for (int d = 0; d < C::DJ; ++d) acc[i][d] *= alpha;
    }
#pragma unroll
    for (int a = 0; a < C::KT; ++a)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[a][u], f, -m[i]));
        s[a][u] = MASKED && !sees(x, i, a, u) ? 0.0f : w;
        l[i] += s[a][u];
      }
  }

  template <bool MASKED, bool AGAIN>
  __device__ __forceinline__ void consume(Step<T, D>& x, Values values) {
    if constexpr (MASKED) {
      // values that no query sees count as zeros (0 times what stands there need not be 0)
#pragma unroll
      for (int e = 0; e < C::KT * 4; ++e) {
        const bool ok = x.key0 + 16 * (e / 4) + 4 * g + e % 4 <= tmax && (x.have >> e) & 1;
#pragma unroll
        for (int w = 0; w < C::VW; ++w) x.v[e][w] = !ok ? 0u : AGAIN ? stand_in<T>(x.v[e][w], values) : x.v[e][w];
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 s[C::KT];
      scores(x, i, s);
      weights<MASKED, AGAIN>(x, i, s, values);
      if constexpr (C::EB == 2) {
        uint32_t hi[2 * C::KT], lo[2 * C::KT];
#pragma unroll
        for (int e = 0; e < 2 * C::KT; ++e) {
          const float w0 = s[e / 2][2 * (e % 2)], w1 = s[e / 2][2 * (e % 2) + 1];
          hi[e] = pack2<T>(w0, w1);
          lo[e] = pack2<T>(w0 - unpack_lo<T>(hi[e]), w1 - unpack_hi<T>(hi[e]));
        }
#pragma unroll
        for (int d = 0; d < C::DJ; ++d) {
          uint32_t vt[2 * C::KT];   // the eight (four) keys' values of one column
#pragma unroll
          for (int e = 0; e < 2 * C::KT; ++e)
            vt[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][d / 2], x.v[2 * e][d / 2], d % 2 ? 0x07060302u : 0x05040100u);
          if constexpr (C::KT == 2) {
            const uint4 va = make_uint4(vt[0], vt[1], vt[2], vt[3]);
            acc[i][d] = mfma32<T>(va, make_uint4(hi[0], hi[1], hi[2], hi[3]), acc[i][d]);
            acc[i][d] = mfma32<T>(va, make_uint4(lo[0], lo[1], lo[2], lo[3]), acc[i][d]);
          } else {
            const u32x2 va = {vt[0], vt[1]};
            acc[i][d] = mfma16<T>(va, (u32x2){hi[0], hi[1]}, acc[i][d]);
            acc[i][d] = mfma16<T>(va, (u32x2){lo[0], lo[1]}, acc[i][d]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < C::KT * 4; ++e)
#pragma unroll
          for (int d = 0; d < C::DJ; ++d)
            acc[i][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[e][d]), s[e / 4][e % 4], acc[i][d], 0, 0, 0);
      }
    }
  }
  template <bool AGAIN>
  __device__ __forceinline__ void step(Step<T, D>& x, Values values) {
    turn(x);
    if constexpr (AGAIN) {
      consume<true, true>(x, values);
    } else {
      const bool full = x.key0 + C::KEYS - 1 <= tmin &&
                        __ballot((x.have & ((1u << (4 * C::KT)) - 1)) != (1u << (4 * C::KT)) - 1) == 0;
      if (full) consume<false, false>(x, kAll);
      else consume<true, false>(x, kAll);
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      m[i] = kLowest;
      l[i] = 0.0f;
#pragma unroll
      for (int d = 0; d < C::DJ; ++d) acc[i][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  template <bool AGAIN, bool STREAM>
  __device__ __forceinline__ void pass(int k0, int k1, Values values) {
    const int last = k0 + (k1 - 1 - k0) / C::KEYS * C::KEYS;   // the last step's first key
    auto at = [&](int n) {
      const int key = k0 + n * C::KEYS;
      return key < last ? key : last;
    };
    pg = page_of(k0);
    // two steps in registers: one arrives while the other is used
    Step<T, D> x[2];
    fetch<STREAM>(x[0], at(0), at(1), true);
    for (int n = 0; k0 + n * C::KEYS < k1; n += 2) {
      fetch<STREAM>(x[1], at(n + 1), at(n + 2), k0 + (n + 1) * C::KEYS < k1);
      step<AGAIN>(x[0], values);
      fetch<STREAM>(x[0], at(n + 2), at(n + 3), k0 + (n + 2) * C::KEYS < k1);
      if (k0 + (n + 1) * C::KEYS < k1) step<AGAIN>(x[1], values);
    }
  }

  // The sums over a row's lanes; zeros for rows whose position is outside the cache.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      l[i] = sum_rows(l[i]);
      if (none >> (kRows * i + c) & 1) {
        m[i] = kLowest;
        l[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < C::DJ; ++d) acc[i][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
  }

  // The rows (bit 16 i + c) whose accumulators are not finite, though the sum of their weights is: where that is not, nor is
  // a weight, and the whole row is NaN.
  __device__ __forceinline__ uint32_t unsound() const {
    uint32_t rows = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      bool bad = false;
#pragma unroll
      for (int d = 0; d < C::DJ; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) bad |= !(fabsf(acc[i][d][u]) < INFINITY);
      const uint64_t w = __ballot(bad), n = __ballot(!(fabsf(l[i]) < INFINITY));
      const uint64_t ww = w | w >> 32, nn = n | n >> 32;
      rows |= (uint32_t)((ww | ww >> 16) & ~(nn | nn >> 16) & 0xffff) << (16 * i);
    }
    return rows;
  }

  // The elements of acc (bit 4 d + u of row set i) that are not zero.
  __device__ __forceinline__ void marks(uint32_t (&bits)[NT]) const {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      bits[i] = 0;
#pragma unroll
      for (int d = 0; d < C::DJ; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) bits[i] |= acc[i][d][u] != 0.0f ? 1u << (4 * d + u) : 0u;
    }
  }
  // Infinities and NaN in the elements that see them.
  __device__ __forceinline__ void mark(const uint32_t (&up)[NT], const uint32_t (&down)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int d = 0; d < C::DJ; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool a = up[i] >> (4 * d + u) & 1, b = down[i] >> (4 * d + u) & 1;
          acc[i][d][u] = a && b ? NAN : a ? INFINITY : b ? -INFINITY : acc[i][d][u];
        }
  }

  // Keys [k0, k1) for the rows of `want`; emit(mask) takes the results of some rows at a time.  stream (one set of rows): by
  // loads that the caches need not keep.
  //
  // A value that is infinite or NaN reaches, in the matrix instructions, rows that do not see its key (as 0 times it), and
  // comes as a sum of two products (which may be inf - inf).  So where a row's result is not finite, its wavefront goes
  // through the keys again: twice with ones for such values and for the weights of what a row sees, which says which elements
  // see +inf, -inf or NaN, and once with zeros for such values (the same sums as if they had been finite).  What is still
  // not finite has passed the range of a float on the way (not float16 values): once more, with weights of at most 2^-24.  Five
  // passes at most, whatever the values are, and the rows that none of it reaches keep their bits.
  template <typename Emit>
  __device__ __forceinline__ void run(int k0, int k1, uint32_t want, bool stream, Emit emit) {
    if (k0 < k1) {
      if (NT == 1 && stream) pass<false, NT == 1>(k0, k1, kAll);
      else pass<false, false>(k0, k1, kAll);
    }
    const uint32_t bad = unsound() & want & ~none;
    finish();
    emit(want & ~bad);
    if (bad == 0) return;
    uint32_t left = bad, up[NT], down[NT];
#pragma unroll 1
    for (int n = kUp; n <= kSmall; ++n) {
      reset();
      pass<true, false>(k0, k1, (Values)n);
      if (n <= kDown) {
        if (n == kUp) marks(up);
        else marks(down);
        continue;
      }
      const uint32_t most = n == kFinite ? unsound() & left : 0;
      finish();
      mark(up, down);
      emit(left & ~most);
      left = most;
      if (left == 0) return;
    }
  }

  // The column of acc[.][d][u] in a row.
  __device__ __forceinline__ int col(int d, int u) const { return MANY ? 16 * d + 4 * g + u : C::DJ * (4 * g + u) + d; }
};

// Many rows, 16 bits: workgroups of four wavefronts with 32 rows each, which share their keys' way through LDS, 64 keys at a
// time, the next 64 on their way there and those behind them in registers.
//
// Bound by instructions: for 32 rows x 32 keys some 115 of the vector units (16 of them exponentials, at a quarter of the rate)
// beside 28 of the matrix cores, two wavefronts to a SIMD.  So what can goes to the matrix cores (the weights' sums, as a
// column of ones) and to LDS (values turned round on the way out, where Share takes 16 permutes); scores are not kept for the
// branch that renews a maximum but made again there; and what the first part of a weight leaves is one dot product.  64 keys
// between two branches, since their chains run beside each other (with 32, three wavefronts to a SIMD spill: 502 us in place
// of 389).
//
// 2 x 12 heads of 64 x 8192 tokens 418 us (493 TFLOP/s of the two products), 8 x 12 x 2048 128, 2 x 8 heads of 128 x 4096 192 (one
// wavefront to a SIMD, whose 512 registers it needs).  In one session 389, 116 and 188 us; 540, 165 and 275 a wavefront a set.
template <typename T, int D>
struct Block : Share<T, D, true, 2, true> {
  using S = Share<T, D, true, 2, true>;
  using C = typename S::C;
  static constexpr int kKeys = 64;
  static constexpr int PR = D * C::EB / 16;                     // 16-byte pieces of a row
  static constexpr int NP = kKeys * PR / (kWaves * kWave);      // of K, and of V, a thread
  static constexpr int LBUF = 2 * kKeys * C::LROW;              // LDS bytes of 64 keys and values
  using S::acc;
  using S::c;
  using S::g;
  using S::kb;
  using S::l;
  using S::lds;
  using S::m;
  using S::none;
  using S::p;
  f32x4 sums[2];        // the weights' sums, by the matrix cores, in every element
  using S::t;
  using S::tab;
  using S::tmax;
  using S::tmin;
  using S::vb;
  struct Pieces {
    uint4 k[NP], v[NP];
    uint32_t ok;        // bit j: keys 32 j ... have a page
  };

  __device__ __forceinline__ Block(const Dense& p_, int b, int h, int row0, char* lds_, bool one = false, int last = -1)
      : S(p_, b, h, row0, lds_, one, last) {
    clear();
  }
  __device__ __forceinline__ void clear() { sums[0] = sums[1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f}; }

  // Requests keys key0 .. key0 + 63 (those past k1 or without a page: some row's, which is not used).
  __device__ __forceinline__ void load(Pieces& x, int key0, int k1) const {
    const int tid = threadIdx.x;
    x.ok = 0;
    int64_t ko[2], vo[2];
    uint32_t last[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = key0 + 32 * j < k1 ? key0 + 32 * j : key0;   // (what stands past k1 no row of the workgroup sees)
      if (tab) {
        const int page = tab[key >> p.blog2];
        const bool ok = page >= 0 && page < p.npages;
        const int64_t to = (ok ? page : 0) * p.pstride;
        const int r = key & ((1 << p.blog2) - 1);
        x.ok |= ok ? 1u << j : 0u;
        ko[j] = to + r * p.kst;
        vo[j] = to + r * p.vst;
        last[j] = 31;
      } else {
        x.ok |= 1u << j;
        ko[j] = key * p.kst;
        vo[j] = key * p.vst;
        last[j] = p.Tk - 1 - key < 31 ? p.Tk - 1 - key : 31;
      }
    }
    const uint32_t ks = (uint32_t)p.kst * C::EB, vs = (uint32_t)p.vst * C::EB;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = tid + kWaves * kWave * i, row = at / PR;
      // (32 rows are 32 PR pieces: a wavefront's are of one half)
      const int j = PR >= 8 ? kWaves * kWave * i / (32 * PR) : __builtin_amdgcn_readfirstlane(row >> 5);
      const uint32_t r = row & 31, rr = r < last[j] ? r : last[j], o = 16 * (at % PR);
      x.k[i] = ldg_piece((const TA_GLOBAL char*)(kb + ko[j]) + (rr * ks + o));
      x.v[i] = ldg_piece((const TA_GLOBAL char*)(vb + vo[j]) + (rr * vs + o));
    }
  }
  static __device__ __forceinline__ uint4 ldg_piece(const TA_GLOBAL char* at) {
    const u32x4_t r = *(const TA_GLOBAL u32x4_t*)at;
    return make_uint4(r.x, r.y, r.z, r.w);
  }
  __device__ __forceinline__ void put(const Pieces& x, char* buf) const {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = threadIdx.x + kWaves * kWave * i;
      char* to = buf + at / PR * C::LROW + 16 * (at % PR);
      *reinterpret_cast<uint4*>(to) = x.k[i];
      *reinterpret_cast<uint4*>(to + kKeys * C::LROW) = x.v[i];
    }
  }

  // The weights of all row sets in place of their scores (0 where masked), a row's running maximum renewed when one of its
  // scores passes it by more than kSlack.  One branch for all sets, so that their products and exponentials stand in one run of
  // instructions.
  // again(i, s) gives the scores of set i anew, for that branch.
  template <bool MASKED, bool AGAIN, typename F>
  __device__ __forceinline__ void weights(const Step<T, D, true>& x, f32x4 (&s)[2][C::KT], Values values, F again) {
    if (AGAIN && values <= kDown) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int a = 0; a < C::KT; ++a)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[i][a][u] = this->sees(x, i, a, u) ? 1.0f : 0.0f;
      return;
    }
    const float shift = AGAIN && values == kSmall ? kLittle : C::kShift;
    const float past = AGAIN && values == kSmall ? kLittle : C::kShift + C::kSlack;
    const float f = fabsf(p.scale) * kLog2e;   // (a negative scale turns q round: the largest score is the largest product)
    float top[2];
    bool some = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = -INFINITY;
#pragma unroll
      for (int a = 0; a < C::KT; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          s[i][a][u] = fmaf(s[i][a][u], f, -m[i]);   // the exponent; masked: -inf
          if (MASKED && !this->sees(x, i, a, u)) s[i][a][u] = -INFINITY;
          top[i] = fmaxf(top[i], s[i][a][u]);
        }
      some |= top[i] > past;
    }
    if (__ballot(some) != 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // only the rows that need it: what a row gives does not depend on the others
        float mx = kLowest;
        f32x4 r[C::KT];
        again(i, r);
#pragma unroll
        for (int a = 0; a < C::KT; ++a)
#pragma unroll
          for (int u = 0; u < 4; ++u) mx = s[i][a][u] != -INFINITY ? fmaxf(mx, r[a][u] * f) : mx;
        mx = max_rows(mx);
        const float mn = max_rows(top[i]) > past ? mx - shift : m[i];
        const float alpha = __builtin_amdgcn_exp2f(m[i] - mn);
        m[i] = mn;
        sums[i] *= alpha;
#pragma unroll
        for (int d = 0; d < C::DJ; ++d) acc[i][d] *= alpha;
#pragma unroll
        for (int a = 0; a < C::KT; ++a)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[i][a][u] = s[i][a][u] != -INFINITY ? fmaf(r[a][u], f, -mn) : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int a = 0; a < C::KT; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[i][a][u] = __builtin_amdgcn_exp2f(s[i][a][u]);
  }

  // 64 keys from LDS; bit j of ok: keys 32 j ... have a page.
  template <bool MASKED, bool AGAIN>
  __device__ __forceinline__ void tile(int key0, uint32_t ok, const char* kl, const char* vl, Values values) {
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    Step<T, D, true> x;
    x.key0 = key0;
    x.have = (ok & 1 ? 0xffu : 0u) | (ok & 2 ? 0xff00u : 0u);
    auto keys = [&]() {
#pragma unroll
      for (int a = 0; a < C::KT; ++a)
#pragma unroll
        for (int e = 0; e < C::KS; ++e)
          x.k[a][e] = *reinterpret_cast<const uint4*>(kl + (16 * a + c) * C::LROW + 64 * e + 16 * g);
    };
    keys();
    f32x4 s[2][C::KT];
#pragma unroll
    for (int i = 0; i < 2; ++i) this->scores(x, i, s[i]);
    weights<MASKED, AGAIN>(x, s, values, [&](int i, f32x4 (&r)[C::KT]) {
      keys();
      this->scores(x, i, r);
    });
    const char* vrow = vl + (4 * g + (c >> 2)) * C::LROW + 8 * (c & 3);
#pragma unroll
    for (int half = 0; half < C::KT / 2; ++half) {
      uint4 hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t hw[4], lw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w0 = s[i][2 * half + e / 2][2 * (e % 2)], w1 = s[i][2 * half + e / 2][2 * (e % 2) + 1];
          hw[e] = pack2<T>(w0, w1);
          lw[e] = rest2<T>(w0, w1, hw[e]);
        }
        hi[i] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
        lo[i] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
      }
      // four keys' values of column 16 d + c: four rows of 16 columns, turned round on their way from LDS
      // (the weights' sums with them: ones in place of values)
      const uint32_t one = __is_same(T, f16_t) ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sums[i] = mfma32<T>(make_uint4(one, one, one, one), hi[i], sums[i]);
        sums[i] = mfma32<T>(make_uint4(one, one, one, one), lo[i], sums[i]);
      }
#pragma unroll
      for (int d = 0; d < C::DJ; ++d) {
        uint32_t v[4];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4_t*)(vrow + (32 * half + 16 * a) * C::LROW + 32 * d)));
          v[2 * a] = r.x;
          v[2 * a + 1] = r.y;
        }
        if constexpr (MASKED) {
          // values that no query sees count as zeros (0 times what stands there need not be 0)
          const int end = ok >> half & 1 ? tmax : -1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 32 * half + 16 * (e / 2) + 4 * g + 2 * (e % 2);
            v[e] = key + 1 <= end ? v[e] : key <= end ? v[e] & 0xffffu : 0u;
            if (AGAIN) v[e] = stand_in<T>(v[e], values);
          }
        }
        const uint4 va = make_uint4(v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][d] = mfma32<T>(va, hi[i], acc[i][d]);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][d] = mfma32<T>(va, lo[i], acc[i][d]);
      }
    }
  }

  // Keys [k0, k1) for the whole workgroup; a wavefront without rows brings its pieces and goes along.
  template <bool AGAIN = false>
  __device__ __forceinline__ void pass(int k0, int k1, bool work, Values values = kAll) {
    if (k0 >= k1) return;
    const int n = (k1 - k0 + kKeys - 1) / kKeys;
    Pieces x;
    if constexpr (AGAIN) {   // (rare: one buffer, and no register for what comes next)
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int key0 = k0 + kKeys * i;
        load(x, key0, k1);
        put(x, lds);
        lds_barrier();
        if (work && key0 <= tmax) tile<true, true>(key0, x.ok, lds, lds + kKeys * C::LROW, values);
        lds_barrier();
      }
      return;
    }
    load(x, k0, k1);
    put(x, lds);
    uint32_t ok = x.ok;
    if (n > 1) load(x, k0 + kKeys, k1);
    lds_barrier();
    for (int i = 0; i < n; ++i) {
      const int key0 = k0 + kKeys * i;
      const char* buf = lds + (i & 1) * LBUF;
      if (work && key0 <= tmax) {
        const char* vals = buf + kKeys * C::LROW;
        if (ok == 3 && key0 + kKeys - 1 <= tmin) tile<false, false>(key0, ok, buf, vals, kAll);
        else tile<true, false>(key0, ok, buf, vals, kAll);
      }
      if (i + 1 < n) {
        put(x, lds + ((i + 1) & 1) * LBUF);
        ok = x.ok;
        if (i + 2 < n) load(x, key0 + 2 * kKeys, k1);
      }
      lds_barrier();
    }
  }

  // As Share::run, by the whole workgroup for any of its rows.
  template <typename Emit>
  __device__ __forceinline__ void run(int k0, int k1, uint32_t want, Emit emit) {
    pass(k0, k1, want != 0);
    sum();
    const uint32_t bad = this->unsound() & want & ~none;
    this->finish();
    emit(want & ~bad);
    if (!__syncthreads_or(bad != 0)) return;
    uint32_t left = bad, up[2], down[2];
#pragma unroll 1
    for (int n = kUp; n <= kSmall; ++n) {
      this->reset();
      clear();
      pass<true>(k0, k1, left != 0, (Values)n);
      if (n <= kDown) {
        if (n == kUp) this->marks(up);
        else this->marks(down);
        continue;
      }
      sum();
      const uint32_t most = n == kFinite ? this->unsound() & left : 0;
      this->finish();
      this->mark(up, down);
      emit(left & ~most);
      left = most;
      if (!__syncthreads_or(left != 0)) return;
    }
  }
  // (a lane's part of a sum: the whole of it, in one lane of the row)
  __device__ __forceinline__ void sum() {
#pragma unroll
    for (int i = 0; i < 2; ++i) l[i] = g == 0 ? sums[i][0] : 0.0f;
  }
};

__device__ __forceinline__ void row_place(const Dense& p, int b, int h, int r, int64_t& out, int64_t& lse) {
  int j, n;
  head_token(p, r, j, n);
  out = b * p.osb + (int64_t)(h * p.G + j) * p.osh + n * p.osn;
  lse = ((int64_t)b * p.Hq + h * p.G + j) * p.Nq + n;
}
__device__ __forceinline__ float lse_of(float m, float l) { return l != 0.0f ? (m + __log2f(l)) * kLn2 : kNegBig; }

// A wavefront a set of 16 NT rows, no split.
template <typename T, int D, bool WIDE, int NT>
__global__ __launch_bounds__(kWaves * kWave, sizeof(T) * D >= 512 ? 1 : 2) void dense_rows_kernel(Dense p) {
  const int64_t per = (p.R + kRows * NT - 1) / (kRows * NT);
  // consecutive sets share their keys: those of one XCD (workgroups go round robin over the 8) are consecutive
  const unsigned n8 = gridDim.x / 8;
  const int64_t wg = (int64_t)(blockIdx.x % 8) * n8 + blockIdx.x / 8;
  const int64_t id = wg * kWaves + __builtin_amdgcn_readfirstlane(wave_id());
  if (id >= per * p.BH) return;
  const int bh = (int)(id / per), row0 = (int)(id % per) * kRows * NT;
  const int b = bh / p.H, h = bh % p.H;
  __shared__ __align__(16) char stage[kWaves * Tile<T, D>::LSTEP];
  Share<T, D, WIDE, NT> s(p, b, h, row0, stage + wave_id() * Tile<T, D>::LSTEP);
  const int left = p.R - row0;
  s.run(0, s.tmax + 1, left >= kRows * NT ? (uint32_t)((1ull << (kRows * NT)) - 1) : (1u << left) - 1, false,
        [&](uint32_t done) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = row0 + kRows * i + s.c;
      if (!(done >> (kRows * i + s.c) & 1)) continue;
      int64_t at, le;
      row_place(p, b, h, r, at, le);
      T* o = reinterpret_cast<T*>(p.out) + at;
      const float inv = s.l[i] != 0.0f ? 1.0f / s.l[i] : 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[s.col(d, u)] = from_f32<T>(s.acc[i][d][u] * inv);
      if (s.g == 0 && p.lse) p.lse[le] = lse_of(s.m[i], s.l[i]);
    }
  });
}

// One set's parts joined: each workgroup has written its part through to memory and counts itself in; the last to arrive joins
// them and resets the counter (no workgroup waits for another).
template <typename T, int D, int kSet>
__device__ __forceinline__ void join_parts(const Dense& p, int b, int h, int row0, int rows, int set, int wg0, int count,
                                           float* smem) {
  const int tid = threadIdx.x;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  TA_DMARK(3);
  uint32_t* cnt = p.cnt + set;
  int* flag = reinterpret_cast<int*>(smem);
  if (tid == 0)
    *flag = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(count - 1);
  __syncthreads();
  const int last = *flag;
  __syncthreads();
  TA_DMARK(4);
  if (!last) return;
  // a thread an element, or several with a share of the parts each where there are few elements: all loads of eight parts at
  // once, so that the parts cost one round trip to memory and not one each
  const float* all = p.ws + (int64_t)wg0 * kSet * (D + 2);
  const int E = rows * D;
  const int groups = E < kWaves * kWave ? kWaves * kWave / E : 1;
  for (int base = 0; base < E; base += kWaves * kWave) {
    const int i = groups > 1 ? tid % E : base + tid, first = groups > 1 ? tid / E : 0;
    const int r = i / D, d = i % D;
    const bool in = i < E && first < groups;
    float M = kLowest, L = 0.0f, a = 0.0f;
    if (in) {
      for (int k0 = first; k0 < count; k0 += 8 * groups) {
        float mk[8], lk[8], vk[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int part = k0 + k * groups;
          const float* q = all + ((int64_t)(part < count ? part : first) * kSet + r) * (D + 2);
          mk[k] = ldgf_dc(q);
          lk[k] = part < count ? ldgf_dc(q + 1) : 0.0f;
          vk[k] = ldgf_dc(q + 2 + d);
        }
        float mn = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) mn = lk[k] != 0.0f ? fmaxf(mn, mk[k]) : mn;
        const float alpha = __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        L *= alpha;
        a *= alpha;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (lk[k] != 0.0f) {
            const float f = __builtin_amdgcn_exp2f(mk[k] - M);
            L = fmaf(lk[k], f, L);
            a = fmaf(vk[k], f, a);
          }
        }
      }
    }
    if (groups > 1) {
      float* mine = smem + 3 * tid;
      mine[0] = M;
      mine[1] = L;
      mine[2] = a;
      __syncthreads();
      if (in && first == 0) {
        for (int k = 1; k < groups; ++k) {
          const float* q = smem + 3 * (tid + k * E);
          if (q[1] != 0.0f) {
            const float mn = fmaxf(M, q[0]);
            const float f0 = __builtin_amdgcn_exp2f(M - mn), f1 = __builtin_amdgcn_exp2f(q[0] - mn);
            M = mn;
            L = fmaf(q[1], f1, L * f0);
            a = fmaf(q[2], f1, a * f0);
          }
        }
      }
    }
    if (in && first == 0) {
      int64_t at, le;
      row_place(p, b, h, row0 + r, at, le);
      reinterpret_cast<T*>(p.out)[at + d] = from_f32<T>(L != 0.0f ? a / L : 0.0f);
      if (d == 0 && p.lse) p.lse[le] = lse_of(M, L);
    }
  }
  TA_DMARK(5);
  if (tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // ready for the next call
}

constexpr int kQuantum = 128;        // keys of one unit of work

// Units of work of sequence b: kQuantum keys each, at least one (its rows are written even where they see nothing).  Lane i of
// a wavefront takes sequence b0 + i; n is the last position that any of its rows sees, -1 for none.
__device__ __forceinline__ int units_of(const Dense& p, int b0, int& n) {
  const int lane = lane_id();
  n = -1;
  if (p.Nq <= 64) {
    if (b0 + lane < p.B) {
      const int32_t* row = p.tq + (b0 + lane) * p.tq_sb;
      for (int i0 = 0; i0 < p.Nq; i0 += 8) {   // eight loads at a time
        int t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = row[i0 + i < p.Nq ? i0 + i : 0];
#pragma unroll
        for (int i = 0; i < 8; ++i) n = t[i] < p.Tk && t[i] > n ? t[i] : n;
      }
    }
  } else {
    for (int k = 0; k < kWave && b0 + k < p.B; ++k) {
      int m = -1;
      for (int i = lane; i < p.Nq; i += kWave) {
        const int t = p.tq[(b0 + k) * p.tq_sb + i];
        m = t < p.Tk && t > m ? t : m;
      }
      m = -min16(-m);
      m = max(max(__builtin_amdgcn_readlane(m, 0), __builtin_amdgcn_readlane(m, 16)),
              max(__builtin_amdgcn_readlane(m, 32), __builtin_amdgcn_readlane(m, 48)));
      n = lane == k ? m : n;
    }
  }
  return b0 + lane < p.B ? (n < kQuantum ? 1 : n / kQuantum + 1) : 0;
}
template <int N>
__device__ __forceinline__ int add_shr(int x) {   // x + that of lane - N of its 16 lanes (0 before the first)
  return x + __builtin_amdgcn_update_dpp(0, x, 0x110 + N, 0xF, 0xF, false);
}
__device__ __forceinline__ int prefix64(int x) {   // sum of lanes 0 .. lane
  x = add_shr<8>(add_shr<4>(add_shr<2>(add_shr<1>(x))));
  const int a = __builtin_amdgcn_readlane(x, 15), b = __builtin_amdgcn_readlane(x, 31), c = __builtin_amdgcn_readlane(x, 47);
  const int row = lane_id() >> 4;
  return x + (row == 0 ? 0 : row == 1 ? a : row == 2 ? a + b : a + b + c);
}

// The sum of x over the wavefront, and its largest.
__device__ __forceinline__ int sum64i(int x) { return __builtin_amdgcn_readlane(prefix64(x), kWave - 1); }
__device__ __forceinline__ int max64i(int x) {
  x = -min16(-x);
  return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
             max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int ceil_div(int a, int b) { return (int)((unsigned)(a + b - 1) / (unsigned)b); }

// The units of every sequence, as each workgroup finds them: those of the first 64 in a lane each, of the others read again.
struct Units {
  const Dense& p;
  int u0, n0;           // units and last position of sequence `lane`
  __device__ __forceinline__ Units(const Dense& p_) : p(p_) { u0 = units_of(p, 0, n0); }
  // f(first sequence, units, last positions) over groups of 64 sequences, until it gives false
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (!f(0, u0, n0)) return;
    for (int b0 = kWave; b0 < p.B; b0 += kWave) {
      int n;
      const int u = units_of(p, b0, n);
      if (!f(b0, u, n)) return;
    }
  }
  // workgroups of one set of every sequence, at `most` units each
  __device__ __forceinline__ int parts(int most) const {
    int s = 0;
    each([&](int, int u, int) {
      s += sum64i(ceil_div(u, most));
      return true;
    });
    return s;
  }
};

// A workgroup's part: keys [k0, k1) (before the end that its rows see) of set `set` of (b, h), part `part` of `count`; wg: its
// place among all, in: the set's among those of its sequence; last: the sequence's last position; units: of all sequences.
struct Part {
  int b, h, set, in, part, count, wg, last, k0, k1, units;
};

// A set gets as many workgroups as its sequence is long, so that sequences of any lengths end together and few long ones fill
// the GPU: the fewest units a workgroup with which all sets together need at most nwg of them (as many as run at once: one
// more costs a round of its own), and a set at most `top` (what joins them is one workgroup).  The grid has nwg or as many as
// there are sets; those that are left over leave at once (false).  sets: of a (sequence, key head).
__device__ __forceinline__ bool find_part(const Dense& p, int sets, int nwg, int top, Part& r) {
  const int per = p.H * sets;                    // sets of a sequence (all units: fewer than 2^31)
  const Units units(p);
  int all = 0, longest = 0;
  units.each([&](int, int u, int) {
    all += sum64i(u);
    longest = max(longest, max64i(u));
    return true;
  });
  const int share = nwg / (per * p.B) < 1 ? 1 : nwg / (per * p.B);   // workgroups that every set can have
  int most = ceil_div(longest, share);
  if (p.B > 1 && share < longest) {
    // sequences shorter than the longest leave workgroups to the others
    int least = ceil_div(all * per, nwg);
    for (int i = 0; i < 6 && least < most; ++i) {
      const int half = (least + most) >> 1;
      if (units.parts(half) * per <= nwg) most = half;
      else least = half + 1;
    }
  }
  if (ceil_div(longest, most) > top) most = ceil_div(longest, top);
  int wg = blockIdx.x;
  if (sets > 1) {
    // sets of one key head share its keys: the workgroups in use next to each other are those of one XCD (they go round robin
    // over the 8; the grid is a multiple of 8)
    const int each = ceil_div(units.parts(most) * per, 8);
    if (wg / 8 >= each) return false;
    wg = wg % 8 * each + wg / 8;
  }
  // its sequence, and the workgroups of that one's sets
  int b = -1, ub = 0, count = 0, start = 0, last = -1;
  units.each([&](int b0, int u, int t) {
    const int n = ceil_div(u, most);
    const int sum = prefix64(n);
    const uint64_t past = __ballot(start + sum * per > wg);
    if (past == 0) {
      start += __builtin_amdgcn_readlane(sum, kWave - 1) * per;
      return true;
    }
    const int i = __ffsll((unsigned long long)past) - 1;
    b = b0 + i;
    ub = __builtin_amdgcn_readlane(u, i);
    count = __builtin_amdgcn_readlane(n, i);
    last = __builtin_amdgcn_readlane(t, i);
    start += (__builtin_amdgcn_readlane(sum, i) - count) * per;
    return false;
  });
  if (b < 0) return false;
  r.b = b;
  r.count = count;
  r.wg = wg;
  r.last = last;
  r.units = all;
  r.in = (wg - start) / count;
  r.part = wg - start - r.in * count;
  r.h = sets > 1 ? r.in / sets : r.in;
  r.set = sets > 1 ? r.in - r.h * sets : 0;
  const int mine = (int)((unsigned)ub / (unsigned)count), more = ub - mine * count;
  const int first = r.part * mine + (r.part < more ? r.part : more);
  r.k0 = first * kQuantum;
  r.k1 = (first + mine + (r.part < more ? 1 : 0)) * kQuantum;
  return true;
}

// Bytes of a cache from which its rows are read by loads that the caches need not keep: what is larger than the last-level
// cache (256 MiB) is not there any more at the next call, and its reads get in each other's way.  Of 32 x 12 queries over
// 32768 keys of 64 (2.8 GB) 489 us with ordinary loads and 439 with these, one stream of 131000 (352 MB) 71.7 and 64.9; three
// caches of 86 MB in turns 23.8 and 25.3.  By what the sequences hold, and at most what the pages or the contiguous cache are:
// 32 x 12 queries over 2000 keys of caches for 65536 (197 MB read) 41.5 us, 50.0 with these.
// Only where one set reads a key: several share them in the second cache.
constexpr int64_t kOnce = (int64_t)256 << 20;

// Workgroups of four wavefronts, each with a share of one set of 16 NT rows (find_part).  once: the cache is of kOnce bytes.
template <typename T, int D, bool WIDE, int NT>
__global__ __launch_bounds__(kWaves * kWave, sizeof(T) * D >= 512 ? 1 : 2) void dense_split_kernel(Dense p, int nwg, int top, bool once) {
  extern __shared__ __align__(16) float smem[];
  constexpr int KEYS = Tile<T, D>::KEYS;
  constexpr int kSet = kRows * NT;
  TA_DMARK(0);
  const int sets = (p.R + kSet - 1) / kSet;      // of a (sequence, key head)
  const int w = __builtin_amdgcn_readfirstlane(wave_id()), tid = threadIdx.x;
  Part at;
  if (!find_part(p, sets, nwg, top, at)) return;
  const int b = at.b, h = at.h, row0 = at.set * kSet;
  const int rows = p.R - row0 < kSet ? p.R - row0 : kSet;
  Share<T, D, WIDE, NT> s(p, b, h, row0, reinterpret_cast<char*>(smem) + w * Tile<T, D>::LSTEP, p.Nq == 1, at.last);
  // its keys, and the equal runs of whole steps of its wavefronts
  const int nkeys = s.tmax + 1;
  const int k0 = at.k0 < nkeys ? at.k0 : nkeys, k1 = at.k1 < nkeys ? at.k1 : nkeys;
  int run = (k1 - k0 + kWaves - 1) / kWaves + KEYS - 1;
  run -= run % KEYS;
  const int from = k0 + w * run < k1 ? k0 + w * run : k1, to = from + run < k1 ? from + run : k1;
  TA_DMARK(1);
  // the four wavefronts' parts, behind their keys: [4][rows][D + 2], first the reference and the sum
  float* const parts = smem + kWaves * Tile<T, D>::LSTEP / 4;
  const bool stream = once && (int64_t)at.units * p.H * (kQuantum * 2 * D * (int)sizeof(T)) >= kOnce;
  s.run(from, to, rows == 32 ? 0xffffffffu : (1u << rows) - 1, stream, [&](uint32_t done) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (!(done >> (kRows * i + s.c) & 1)) continue;
      float* part = parts + (w * rows + kRows * i + s.c) * (D + 2);
      if (s.g == 0) {
        part[0] = s.m[i];
        part[1] = s.l[i];
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int u = 0; u < 4; ++u) part[2 + s.col(d, u)] = s.acc[i][d][u];
    }
  });
  TA_DMARK(2);
  __syncthreads();
  float* ws = p.ws + (int64_t)at.wg * kSet * (D + 2);
  for (int i = tid; i < rows * D; i += kWaves * kWave) {
    const int r = i / D, d = i % D;
    float M = kLowest, L = 0.0f, a = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float* q = parts + (k * rows + r) * (D + 2);
      if (q[1] != 0.0f) M = fmaxf(M, q[0]);
    }
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float* q = parts + (k * rows + r) * (D + 2);
      const float f = q[1] != 0.0f ? __builtin_amdgcn_exp2f(q[0] - M) : 0.0f;
      if (q[1] != 0.0f) {
        L = fmaf(q[1], f, L);
        a = fmaf(q[2 + d], f, a);
      }
    }
    if (at.count == 1) {
      int64_t to, le;
      row_place(p, b, h, row0 + r, to, le);
      reinterpret_cast<T*>(p.out)[to + d] = from_f32<T>(L != 0.0f ? a / L : 0.0f);
      if (d == 0 && p.lse) p.lse[le] = lse_of(M, L);
    } else {
      stgf_dc(ws + r * (D + 2) + 2 + d, a);
      if (d == 0) {
        stgf_dc(ws + r * (D + 2), M);
        stgf_dc(ws + r * (D + 2) + 1, L);
      }
    }
  }
  if (at.count > 1) join_parts<T, D, kSet>(p, b, h, row0, rows, b * p.H * sets + at.in, at.wg - at.part, at.count, smem);
}

// Workgroups of four wavefronts with 32 rows each of a set of 128, all over the same keys (Block).  nwg 0: one a set, the
// longest sets first: 2 x 12 heads x 8192 tokens 403 us so, 470 a key head at a time.  Else a set's keys are split (find_part)
// and its parts joined by a launch of its own (dense_join_kernel): 128 rows are too many for the workgroup that comes last.  2
// x 12 heads x 256 rows over 8000 keys 50 us (60 by sets of 32 rows; 88 and more with the last workgroup's join).
constexpr int kBlock = kWaves * 2 * kRows;
constexpr int kManyRows = 96;
// (Heads of 32: three wavefronts to a SIMD, 2 x 12 heads x 8192 tokens 276 us; two 329.  What spills for it is in the passes
// after the first.)
template <typename T, int D>
__global__ __launch_bounds__(kWaves * kWave, D == 128 ? 1 : D == 64 ? 2 : 3) void dense_block_kernel(Dense p, int nwg) {
  using S = Block<T, D>;
  __shared__ __align__(16) char smem[2 * S::LBUF];
  const int sets = (p.R + kBlock - 1) / kBlock, w = __builtin_amdgcn_readfirstlane(wave_id());
  Part at;
  if (nwg > 0) {
    if (!find_part(p, sets, nwg, 1 << 20, at)) return;
    if (at.part == 0 && threadIdx.x == 0) {
      p.heads[(int64_t)at.b * p.H * sets + at.in] = make_int2(at.wg, at.count);
    }
  } else {
    // (the last rows of a prompt see the most; the sets of a key head go to one XCD where there are a multiple of 8 of these)
    const int rank = blockIdx.x / p.BH, bh = blockIdx.x - rank * p.BH, b = bh / p.H;
    at = Part{b, bh - b * p.H, sets - 1 - rank, 0, 0, 1, 0, -1, 0, 0x7fffffff};
  }
  const int b = at.b, h = at.h, row0 = at.set * kBlock + w * 2 * kRows;
  S s(p, b, h, row0, smem);
  int* const ends = reinterpret_cast<int*>(smem);
  if (s.lane == 0) ends[w] = s.tmax + 1;
  __syncthreads();
  const int nkeys = __builtin_amdgcn_readfirstlane(max(max(ends[0], ends[1]), max(ends[2], ends[3])));
  __syncthreads();
  const int k0 = at.k0 < nkeys ? at.k0 : nkeys, k1 = at.k1 < nkeys ? at.k1 : nkeys;
  const int left = p.R - row0;
  const uint32_t want = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1 : 0u;
  const bool whole = at.count == 1;
  float* const part = p.ws + ((int64_t)at.wg * kBlock + w * 2 * kRows) * (D + 4);
  s.run(k0, k1, want, [&](uint32_t done) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = kRows * i + s.c;
      if (!(done >> r & 1)) continue;
      if (whole) {
        int64_t to, le;
        row_place(p, b, h, row0 + r, to, le);
        T* o = reinterpret_cast<T*>(p.out) + to;
        const float inv = s.l[i] != 0.0f ? 1.0f / s.l[i] : 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int u = 0; u < 4; ++u) o[s.col(d, u)] = from_f32<T>(s.acc[i][d][u] * inv);
        if (s.g == 0 && p.lse) p.lse[le] = lse_of(s.m[i], s.l[i]);
      } else {
        float* o = part + r * (D + 4);
        if (s.g == 0) *reinterpret_cast<float2*>(o) = make_float2(s.m[i], s.l[i]);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(o + 4 + s.col(d, 0)) = s.acc[i][d];
      }
    }
  });
}

// The parts of dense_block_kernel's rows joined, D / 4 threads a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void dense_join_kernel(Dense p) {
  constexpr int kPer = 256 / (D / 4);            // rows a workgroup
  const int sets = (p.R + kBlock - 1) / kBlock;
  const int per = (p.R + kPer - 1) / kPer;
  const int bh = blockIdx.x / per, row = (blockIdx.x - bh * per) * kPer + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  if (row >= p.R) return;
  const int b = bh / p.H, h = bh - b * p.H, set = row / kBlock;
  const int2 head = p.heads[(int64_t)bh * sets + set];
  if (head.y == 1) return;                       // (written by its only workgroup)
  const float* q = p.ws + ((int64_t)head.x * kBlock + row - set * kBlock) * (D + 4);
  const int64_t step = (int64_t)kBlock * (D + 4);
  float M = kLowest, L = 0.0f;
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = 0; k0 < head.y; k0 += 8) {
    float2 ml[8];
    f32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* x = q + (k0 + k < head.y ? k0 + k : 0) * step;
      ml[k] = *reinterpret_cast<const float2*>(x);
      v[k] = *reinterpret_cast<const f32x4*>(x + 4 + d);
      if (k0 + k >= head.y) ml[k].y = 0.0f;
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < 8; ++k) mn = ml[k].y != 0.0f ? fmaxf(mn, ml[k].x) : mn;
    const float alpha = __builtin_amdgcn_exp2f(M - mn);
    M = mn;
    L *= alpha;
    a *= alpha;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (ml[k].y != 0.0f) {
        const float f = __builtin_amdgcn_exp2f(ml[k].x - M);
        L = fmaf(ml[k].y, f, L);
#pragma unroll
        for (int u = 0; u < 4; ++u) a[u] = fmaf(v[k][u], f, a[u]);
      }
    }
  }
  int64_t at, le;
  row_place(p, b, h, row, at, le);
#pragma unroll
  for (int u = 0; u < 4; ++u) reinterpret_cast<T*>(p.out)[at + d + u] = from_f32<T>(L != 0.0f ? a[u] / L : 0.0f);
  if (d == 0 && p.lse) p.lse[le] = lse_of(M, L);
}

template <typename T, int D, bool WIDE, int NT>
int launch_dense(const Dense& p, int nsplit, hipStream_t st) {
  const dim3 blk(kWaves * kWave);
  const int64_t per = (p.R + kRows * NT - 1) / (kRows * NT), sets = p.BH * per;
  if (nsplit == 1) {
    const int64_t wgs = ((sets + kWaves - 1) / kWaves + 7) / 8 * 8;
    hipLaunchKernelGGL((dense_rows_kernel<T, D, WIDE, NT>), dim3((unsigned)wgs), blk, 0, st, p);
    return check_launch("dense_rows_kernel");
  }
  const int rows = p.R < kRows * NT ? p.R : kRows * NT;
  const size_t stage = kWaves * Tile<T, D>::LSTEP, parts = (size_t)kWaves * rows * (D + 2), join = 3 * kWaves * kWave;
  const int nwg = nsplit / kWaves;
  const int64_t wgs = nwg < sets ? sets : nwg;
  // (rows of 64, one set of 131000 keys: a row 128 parts 17.6 us, 256 parts 19.5; eight rows 64 parts 32 us, 256 parts 57)
  const int top = rows > 10 ? 24 : 256 / rows;
  const dim3 grid((unsigned)(per > 1 ? (wgs + 7) / 8 * 8 : wgs));
  const size_t lds = stage + (parts > join ? parts : join) * sizeof(float);
  const int64_t bytes = (int64_t)sizeof(T) * (p.ptab ? p.npages * p.pstride : (int64_t)p.BH * p.Tk * 2 * D);
  const bool once = NT == 1 && per == 1 && bytes >= kOnce;
  hipLaunchKernelGGL((dense_split_kernel<T, D, WIDE, NT>), grid, blk, lds, st, p, nwg, top, once);
  return check_launch("dense_split_kernel");
}

// Two tiles of rows a wavefront where there are more rows than one takes: they share the keys' way into the registers.  Not
// with float32 rows (their matrix instructions take longer than that way) nor heads of 128 (registers).
template <typename T, int D>
constexpr int two_tiles() { return sizeof(T) == 2 && D < 128 ? 2 : 1; }

template <typename T, int D>
int block_dense(const Dense& p, int nsplit, hipStream_t st) {
  const int64_t sets = p.BH * (((int64_t)p.R + kBlock - 1) / kBlock);
  const int nwg = nsplit > kWaves ? nsplit / kWaves : 0;
  const int64_t wgs = nwg < sets ? sets : nwg;
  const dim3 grid((unsigned)(nwg > 0 ? (wgs + 7) / 8 * 8 : wgs)), blk(kWaves * kWave);
  hipLaunchKernelGGL((dense_block_kernel<T, D>), grid, blk, 0, st, p, nwg);
  const int rc = check_launch("dense_block_kernel");
  if (rc != TA_OK || nwg <= sets) return rc;     // (no set has more than one)
  constexpr int kPer = 256 / (D / 4);
  const int64_t joins = p.BH * (((int64_t)p.R + kPer - 1) / kPer);
  hipLaunchKernelGGL((dense_join_kernel<T, D>), dim3((unsigned)joins), dim3(256), 0, st, p);
  return check_launch("dense_join_kernel");
}

template <typename T, int D, bool WIDE>
int rows_dense(const Dense& p, int nsplit, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && WIDE && D >= 32)
    // (a workgroup a set of 128 rows; 24 heads x 1024 tokens, 192 workgroups, 28.8 us and 31.1 a wavefront a set, 8 heads of
    // 128 x 2048, 128 of them, 89 and 78; caches of 128 keys 12.8 and 10.7, of 512 20.0 and 24.0; 64 rows over 4000 keys 94
    // and 114)
    if (nsplit != kWaves && p.R >= kManyRows && p.Tk >= 512 &&
        (nsplit > 1 || p.BH * (((int64_t)p.R + kBlock - 1) / kBlock) >= 192))
      return block_dense<T, D>(p, nsplit, st);
  if constexpr (two_tiles<T, D>() == 2)
    if (p.R > kRows) return launch_dense<T, D, WIDE, 2>(p, nsplit, st);
  return launch_dense<T, D, WIDE, 1>(p, nsplit, st);
}

template <typename T>
int dispatch_dense(const Dense& p, int nsplit, hipStream_t st) {
  const bool wide = p.ptab == nullptr || p.blog2 >= 5;   // a step's 32 keys in one run of rows
#define TA_DENSE(DD) return wide ? rows_dense<T, DD, true>(p, nsplit, st) : rows_dense<T, DD, false>(p, nsplit, st)
  switch (p.D) {
    case 16: TA_DENSE(16);
    case 32: TA_DENSE(32);
    case 64: TA_DENSE(64);
    default: TA_DENSE(128);
  }
#undef TA_DENSE
}

}  // namespace
}  // namespace ta

using namespace ta;

namespace ta {
namespace {
// Counters and sets of whole tiles of 32 rows (16 where there are no more), whichever the kernels take.
int64_t dense_sets(int B, int Hq, int H, int Nq) {
  const int64_t R = (int64_t)(Hq / H) * Nq;
  return (int64_t)B * H * (R <= 16 ? 1 : (R + 31) / 32 * 2);
}
// Bytes of the counters, and of the heads of a quarter as many sets or fewer behind them.
int64_t counter_bytes(int64_t sets) { return (sets * 4 + 255) / 256 * 256 * 2; }
}  // namespace
}  // namespace ta

extern "C" int64_t ta_dense_attn_workspace_size(int B, int Hq, int H, int Nq, int D, int nsplit) {
  if (B <= 0 || H <= 0 || Hq <= 0 || Nq <= 0 || nsplit <= 4) return 0;
  const int64_t sets = dense_sets(B, Hq, H, Nq);
  // counters; heads; a part for each workgroup and each set, of 16 rows, or of 32 or 128 for fewer sets
  const int64_t R = (int64_t)(Hq / H) * Nq, rows = R < kManyRows ? 32 : kBlock;
  const int64_t all = R < kManyRows ? sets * 16 : (int64_t)B * H * ((R + kBlock - 1) / kBlock * kBlock);
  return counter_bytes(sets) + (all + nsplit / 4 * rows) * (D + 4) * 4;
}

extern "C" int ta_dense_attn_fwd(const void* q, const void* k, const void* v, int dtype, int64_t qsb, int64_t qsh,
                                 int64_t qsn, int64_t ksb, int64_t ksh, int64_t kst, int64_t vsb, int64_t vsh, int64_t vst,
                                 int B, int Hq, int H, int Nq, int D, int Tk, const int32_t* tq, int64_t tq_sb, float scale,
                                 void* out, int64_t osb, int64_t osh, int64_t osn, float* lse, int nsplit, float* ws,
                                 int64_t ws_bytes, const ta_kv_pages* pages, void* stream) {
  if (dtype != TA_F32 && dtype != TA_F16 && dtype != TA_BF16) {
    set_error("ta_dense_attn_fwd: unknown dtype");
    return TA_ERR_ARG;
  }
  if (D != 16 && D != 32 && D != 64 && D != 128) {
    set_error("ta_dense_attn_fwd: head dim must be 16, 32, 64 or 128");
    return TA_ERR_UNSUPPORTED;
  }
  if (B < 0 || H < 1 || Hq < 1 || Hq % H || Nq < 0 || Tk < 1) {
    set_error("ta_dense_attn_fwd: bad sizes (query heads a multiple of the key heads)");
    return TA_ERR_ARG;
  }
  if (nsplit < 1 || (nsplit > 1 && nsplit % 4) || nsplit > 8192) {
    set_error("ta_dense_attn_fwd: nsplit must be 1 or a multiple of 4, at most 8192");
    return TA_ERR_ARG;
  }
  if (pages && (pages->table == nullptr || pages->num_pages <= 0 || pages->block_log2 < 1 || pages->block_log2 > 14)) {
    set_error("ta_dense_attn_fwd: bad page description");
    return TA_ERR_ARG;
  }
  if (B == 0 || Nq == 0) return TA_OK;
  if (q == nullptr || k == nullptr || v == nullptr || tq == nullptr || out == nullptr) {
    set_error("ta_dense_attn_fwd: a missing pointer");
    return TA_ERR_ARG;
  }
  // (a stride of a dimension of one is never a step)
  if (B == 1) qsb = ksb = vsb = 0;
  if (Hq == 1) qsh = 0;
  if (H == 1) ksh = vsh = 0;
  if (Nq == 1) qsn = 0;
  if (Tk == 1 && !pages) kst = vst = 0;
  const int sz = dtype == TA_F32 ? 4 : 2;
  const int64_t bits = (int64_t)((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) | (qsb | qsh | qsn | kst | vst) * sz |
                       (pages ? pages->page_stride * sz : (ksb | ksh | vsb | vsh) * sz);
  if (bits % 16) {
    set_error("ta_dense_attn_fwd: q, K and V rows must be 16-byte aligned");
    return TA_ERR_ARG;
  }
  const int64_t R = (int64_t)(Hq / H) * Nq;
  const int64_t sets = dense_sets(B, Hq, H, Nq);
  if (R > (1 << 30) || sets > (1 << 30) || Tk > 0x7fffffff - 4096 ||
      (nsplit > 1 && sets * ((Tk + 127) / 128) > 0x7fffffffLL)) {
    set_error("ta_dense_attn_fwd: too large");
    return TA_ERR_UNSUPPORTED;
  }
  if (kst < 0 || vst < 0 || kst * sz * 32 > 0x7fffffffLL || vst * sz * 32 > 0x7fffffffLL) {
    set_error("ta_dense_attn_fwd: row strides from 0 to 64 MiB");
    return TA_ERR_UNSUPPORTED;
  }
  const int64_t need = ta_dense_attn_workspace_size(B, Hq, H, Nq, D, nsplit);
  if (need > 0 && (ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256)) {
    set_error("ta_dense_attn_fwd: workspace missing, too small or not 256-byte aligned");
    return TA_ERR_WORKSPACE;
  }
  Dense p{q, qsb, qsh, qsn, k, ksb, ksh, kst, v, vsb, vsh, vst, Hq, H, Hq / H, Nq, D, Tk, tq, tq_sb, scale, out, osb, osh,
          osn, lse};
  if (pages) {
    p.ptab = pages->table;
    p.pt_sb = pages->sb;
    p.pt_sh = pages->sh;
    p.pstride = pages->page_stride;
    p.npages = pages->num_pages;
    p.blog2 = pages->block_log2;
  }
  p.BH = B * H;
  p.R = (int)R;
  p.B = B;
  if (need > 0) {
    p.cnt = reinterpret_cast<uint32_t*>(ws);
    p.heads = reinterpret_cast<int2*>(reinterpret_cast<char*>(ws) + counter_bytes(sets) / 2);
    p.ws = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + counter_bytes(sets));
  }
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TA_F32) return dispatch_dense<float>(p, nsplit, st);
  if (dtype == TA_F16) return dispatch_dense<f16_t>(p, nsplit, st);
  return dispatch_dense<bf16_t>(p, nsplit, st);
}

TA_TRACE_EXPORTS
