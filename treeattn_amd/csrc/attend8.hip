// Sparse softmax attention over a cache of 8-bit pages (kv8.hpp): the selected leaf blocks, the own block and the
// static keys of each query, as attend.hip has it over caches in the model's type.
//
// For key j of a page with scales (sk, sv), k_j = sk * k8_j and v_j = sv * v8_j:
//   s_j = scale * sk * (q . k8_j),  out = sum_j e^(s_j - M) sv * v8_j / sum_j e^(s_j - M)
// so a page's scales cost one multiplication per key, not per element.  Keys of the block that the tail holds are read
// from there, unrounded.  Sums, maxima and the accumulators are float32; the output is rounded once.
//
// One pass over the keys with a running maximum and sum.  A key row is D bytes, so D / 16 lanes hold a row, a load brings 64 *
// 16 / D keys' K or V, and a chunk is two of each; four chunks are in flight.  No matrix instruction: one query a page
// leaves 15 of a tile's 16 rows idle, and the vector units are busy 30 % of a launch of many queries.
//
// Many queries are bound by the bytes, 2 D a key: 32 x 12 queries over 2048 + 32 keys of 64 (102 MB) take 25 us, 4.1 TB/s; as
// many workgroups that do nothing but read such pages take 21 (the unquantised cache's 204 MB take 40.5 us).  Few queries
// have one wavefront to a SIMD, so that nothing runs beside its waits and its instructions: 12 queries over 8192 keys of 64
// by 64 wavefronts each take 12.8 us (12.7 MB), of which a wavefront waits 52 % -- a chain of round trips: position and leaf
// ids, page table, scales with the keys, the workgroups' partials and their join -- and issues instructions 42 %: its key
// list, which every wavefront makes for itself, four or five chunks of keys and as many requests past the last key, the sums
// across lanes (14.1 us with the tail's rows requested behind the keys, the page reads behind the count of the valid leaves
// and sums across lanes by shuffles).
//
// Reference functions replaced: engine.py:107-119 (decode attention).
#include "attn.hpp"
#include "kv8.hpp"

namespace ta {
namespace {

constexpr int kWaves = 4;
constexpr float kLowest = -3.4028235e38f;

struct Attn8 {
  const void* q;
  int64_t qsb, qsh, qsn;
  Kv8 c;
  int H, Nq;
  const int32_t* tq;
  int64_t tq_sb;
  const int32_t* ids;
  const uint8_t* vld;
  const int32_t* n_tree;
  int wl, Lw;
  float scale;
  int gsplit;
  void* out;
  int64_t osb, osh, osn;
  float* lse;
  float* keys;
  float* ws;
  uint32_t* cnt;
  const int32_t* nb_id;
  const uint8_t* nb_ok;
  int nb_S;
};

// Entries of a wavefront's key list: the tree leaves, the neighbour leaves, the own block and at most 32 static keys.
__host__ __device__ constexpr int list8_cap(int wl, int nb_S) { return ((wl + 3) & ~3) + ((nb_S + 3) & ~3) + 36; }
// LDS words of a wavefront: per entry its first row, its leaf id and its two scales.
__host__ __device__ constexpr int list8_ints(int cap) { return 4 * cap; }

// The larger of x over the wavefront, in every lane.
__device__ __forceinline__ float max64(float x) {
  x = fmaxf(x, dpp_f<0xB1>(x));
  x = fmaxf(x, dpp_f<0x4E>(x));
  x = fmaxf(x, dpp_f<0x141>(x));
  x = fmaxf(x, dpp_f<0x140>(x));
  // (with one register in both places the exchange gives its halves, each spread over the lanes)
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum64(float x) {
  x = group_sum<16>(x);
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Sums of acc over the lanes that share lane % LPR.  Each exchange of halves leaves a lane half as many sums: lane l ends
// with elements 8 * (l / 32) + 4 * (l / 16 % 2) + 0 .. 3 of its 16 in out, the same in all lanes of its 16 that share l % LPR.
template <int LPR>
__device__ __forceinline__ void sum_rows(float (&acc)[16], float (&out)[4]) {
  float h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i + 8]), false, false);
    h[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[i]), __float_as_uint(h[i + 4]), false, false);
    float x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    if constexpr (LPR <= 8) x += dpp_f<0x128>(x);   // rotations within 16 lanes
    if constexpr (LPR <= 4) x += dpp_f<0x124>(x);
    if constexpr (LPR <= 2) x += dpp_f<0x122>(x);
    if constexpr (LPR <= 1) x += dpp_f<0x121>(x);
    out[i] = x;
  }
}

// SPLIT: the four wavefronts of a workgroup, and p.gsplit workgroups, share one query; else a wavefront has a query of
// its own.
template <typename T, int D, bool SPLIT>
__global__ __launch_bounds__(kWaves * kWave) void attn8_kernel(Attn8 p) {
  extern __shared__ __align__(16) float smem_f[];
  constexpr int E = 16;              // elements of a row per lane: 16 bytes of e4m3
  constexpr int LPR = D / E;         // lanes per key row
  constexpr int RPI = kWave / LPR;   // key rows per load instruction
  constexpr int NL = 2;              // load instructions per chunk
  constexpr int KPC = NL * RPI;      // keys per chunk
  constexpr int PF = 4;              // chunks in flight
  const int lane = lane_id(), w = wave_id();
  int n, g = 0;
  if constexpr (SPLIT) {
    n = blockIdx.x / p.gsplit;
    g = blockIdx.x % p.gsplit;
  } else {
    n = blockIdx.x * kWaves + w;
    if (n >= p.Nq) return;
  }
  const int bh = blockIdx.y;
  const int b = bh / p.H, h = bh % p.H;
  const int64_t qi = (int64_t)bh * p.Nq + n;
  const Kv8& c = p.c;
  const int leaf = 1 << c.blog2, mask = leaf - 1;
  const int nblk = (c.tcap + leaf - 1) >> c.blog2;
  const int cap = list8_cap(p.wl, p.nb_S);
  int32_t* s_row = reinterpret_cast<int32_t*>(smem_f) + w * list8_ints(cap);
  int32_t* s_id = s_row + cap;
  float2* s_sc = reinterpret_cast<float2*>(s_id + cap);
  const int rg = lane / LPR;
  const int ds = (lane % LPR) * E;

  // everything whose place is known at once: the query, its position, the block in the tail, the selected leaves
  const int32_t* idr = p.ids + qi * p.wl;
  const uint8_t* vr = p.vld + qi * p.wl;
  const int32_t* trow = c.table + b * c.sb + h * c.sh;
  int t = p.tq[b * p.tq_sb + n];
  const int held = c.tail_block[b * c.tb_sb + h];
  const int nt = p.n_tree ? p.n_tree[qi] : p.wl;
  const int id0 = lane < p.wl ? idr[lane] : -1;
  const bool v0 = lane < p.wl && vr[lane] != 0;
  float qv[E];
  load_row_g<T, E>(reinterpret_cast<const T*>(p.q) + b * p.qsb + h * p.qsh + n * p.qsn + ds, qv);

  if (t < 0 || t >= c.tcap) t = -1;   // out of range: attend nothing
  const int own = t < 0 ? -1 : t >> c.blog2;
  const int lb = t < 0 ? 0 : own << c.blog2;
  const int tr = t & mask;
  // Page reads: the first 64 leaves'; the static keys' [0, t, t-1, ..., t-Lw+1] by lanes 0 .. Lw and the own block's by lane
  // Lw + 1.  The first row of the block's page, -1 where it has none, lies outside the table or is the one in the tail
  // (whose keys are added from there).
  auto first_row = [&](int id) {
    int row = -1;
    if (id >= 0 && id < nblk && id != held) {
      const int pg = c.page(trow, id);
      if (pg >= 0) row = pg << (c.blog2 + 1);
    }
    return row;
  };
  int pe = -1;
  if (lane <= p.Lw && t >= 0) pe = lane == 0 ? 0 : t - (lane - 1);
  const int pb = lane == p.Lw + 1 ? own : (pe >= 0 ? pe >> c.blog2 : -1);
  const int row0 = first_row(id0);
  const int srow = first_row(pb);

  // The block in the tail: its first rows are requested here, behind the page reads.
  const bool mine = held == own;
  const int stride = SPLIT ? p.gsplit * kWaves : 1;
  const int first = SPLIT ? g * kWaves + w : 0;
  const int trows = t >= 0 && held >= 0 ? (mine ? tr + 1 : leaf) : 0;
  const T* tk = reinterpret_cast<const T*>(c.tail) + b * c.tail_sb + h * c.tail_sh + ds;
  float tkv[E], tvv[E];
  auto load_tail = [&](int r) {
    const int64_t rc = r < trows ? r : 0;
    load_row_g<T, E>(tk + rc * D, tkv);
    load_row_g<T, E>(tk + (int64_t)leaf * D + rc * D, tvv);
  };
  if (first * RPI < trows) load_tail(first * RPI + rg);

  int nv = __popcll(__ballot(v0));
  for (int i0 = kWave; i0 < p.wl; i0 += kWave) nv += __popcll(__ballot(i0 + lane < p.wl && vr[i0 + lane] != 0));
  int nused = t < 0 ? 0 : (nv < nt ? nv : (nt > 0 ? nt : 0));
  bool all = __ballot(lane < nused && id0 == held && held >= 0) != 0;   // the tail's block is among the selected ones
  if (lane < nused) {
    s_id[lane] = id0;
    s_row[lane] = row0;
  }
  for (int i0 = kWave; i0 < nused; i0 += kWave) {
    const int i = i0 + lane;
    const int id = i < nused ? idr[i] : -1;
    if (i < nused) {
      s_id[i] = id;
      s_row[i] = first_row(id);
    }
    all |= __ballot(i < nused && id == held && held >= 0) != 0;
  }
  wave_sync();
  if (p.nb_S > 0 && t >= 0) {
    // a matched neighbour slot joins when its block is complete before the own block, is not one of the tree leaves
    // and no earlier matched slot holds the same one (fastseg.py:376-381)
    const bool in = lane < p.nb_S;
    const int id = in ? p.nb_id[qi * p.nb_S + lane] : -1;
    const bool cand = in && p.nb_ok[qi * p.nb_S + lane] != 0 && id >= 0;
    bool keep = cand && id < own;
    for (int i = 0; i < nused; ++i)
      if (s_id[i] == id) keep = false;
    const uint64_t cm = __ballot(cand);
    for (int s2 = 0; s2 < p.nb_S; ++s2) {
      const int o = __shfl(id, s2, kWave);
      if (((cm >> s2) & 1) && s2 < lane && o == id) keep = false;
    }
    const uint64_t km = __ballot(keep);
    if (keep) {
      const int slot = nused + __popcll(km & ((1ull << lane) - 1));
      s_id[slot] = id;
      s_row[slot] = first_row(id);
    }
    all |= __ballot(keep && id == held) != 0;
    nused += __popcll(km);
    wave_sync();
  }
  // static keys: those >= 0, outside the own block, whose block is not used, the sink once
  bool keep = pe >= 0 && pe < lb && !(lane > 0 && pe == 0);
  if (keep) {
    const int lf = pe >> c.blog2;
    for (int i = 0; i < nused; ++i)
      if (s_id[i] == lf) keep = false;
  }
  const uint64_t bal = __ballot(keep);
  const int next = __popcll(bal);
  const int nblocks = nused + (t < 0 ? 0 : 1);   // the own block is the last of the blocks
  if (keep) s_row[nblocks + __popcll(bal & ((1ull << lane) - 1))] = srow < 0 ? -1 : srow + (pe & mask);
  if (t >= 0 && lane == p.Lw + 1) s_row[nused] = srow;
  wave_sync();
  const int nl = nblocks << c.blog2;    // keys of the blocks (the own block's past t masked), then the static ones
  const int N8 = nl + next;

  const char* kb = reinterpret_cast<const char*>(c.pool) + ds;
  const int64_t vofs = (int64_t)leaf * D;
  const int nchunks = (N8 + KPC - 1) / KPC;

  struct Chunk {
    uint4 k[NL], v[NL];
    int e[NL];     // entry of the key, -1: none
  };
  auto fetch = [&](int ci, Chunk& x) {
    int row[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int key = ci * KPC + i * RPI + rg;
      const bool blk = key < nl;
      const int kc = key < N8 ? key : 0;
      const int e = blk ? kc >> c.blog2 : (key < N8 ? nblocks + (kc - nl) : 0);
      const int rr = blk ? kc & mask : 0;
      const int r0 = N8 > 0 ? s_row[e] : -1;
      const bool ok = key < N8 && r0 >= 0 && !(blk && e == nused && rr > tr);
      x.e[i] = ok ? e : -1;
      row[i] = ok ? r0 + rr : 0;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const char* a = kb + (int64_t)row[i] * D;
      x.k[i] = ldg16(a);
      x.v[i] = ldg16(a + vofs);
    }
  };

  float m = kLowest, l = 0.0f;
  float acc[E];
#pragma unroll
  for (int d = 0; d < E; ++d) acc[d] = 0.0f;
  // NK keys of this lane's row group: scores (already scaled) and their values
  auto rescale = [&](float mn) {
    const float alpha = __expf(m - mn);
#pragma unroll
    for (int d = 0; d < E; ++d) acc[d] *= alpha;
    l *= alpha;
    m = mn;
  };
  auto consume = [&](const Chunk& x) {
    float sc[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      float kv[E];
      e4m3_x16(x.k[i], kv);
      float d0 = 0.0f;
#pragma unroll
      for (int d = 0; d < E; ++d) d0 = fmaf(qv[d], kv[d], d0);
      sc[i] = d0;
    }
    float cm = kLowest, vs[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const float2 s = s_sc[x.e[i] < 0 ? 0 : x.e[i]];
      sc[i] = group_sum<LPR>(sc[i]) * (s.x * p.scale);
      vs[i] = s.y;
      if (x.e[i] >= 0) cm = fmaxf(cm, sc[i]);
    }
    rescale(fmaxf(m, cm));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const float pw = x.e[i] >= 0 ? __expf(sc[i] - m) : 0.0f;
      l += pw;
      const float pv = pw * vs[i];
      float vv[E];
      e4m3_x16(x.v[i], vv);
      if (x.e[i] >= 0) {
#pragma unroll
        for (int d = 0; d < E; ++d) acc[d] = fmaf(pv, vv[d], acc[d]);
      }
    }
  };

  // keys of the tail: all its rows when it is selected, those up to t when it is the own block, else its static keys
  auto consume_tail = [&](int r) {
    const int pos = (held << c.blog2) + r;
    const bool ok = r < trows && (mine || all || (held < own && (pos == 0 || pos > t - p.Lw)));
    float s = 0.0f;
#pragma unroll
    for (int d = 0; d < E; ++d) s = fmaf(qv[d], tkv[d], s);
    s = group_sum<LPR>(s) * p.scale;
    rescale(fmaxf(m, ok ? s : kLowest));
    if (ok) {
      const float pw = __expf(s - m);
      l += pw;
#pragma unroll
      for (int d = 0; d < E; ++d) acc[d] = fmaf(pw, tvv[d], acc[d]);
    }
  };
  auto tail = [&]() {
    for (int r0 = first * RPI; r0 < trows; r0 += stride * RPI) {
      if (r0 > first * RPI) load_tail(r0 + rg);
      consume_tail(r0 + rg);
    }
  };

  if (nchunks > 0) {
    // The entries' scales: requested with the first keys, so that they are no round trip of their own, and before them,
    // since loads return in order (lists of more than 64 entries take the rest at once).
    const int entries = nblocks + next;
    auto scales = [&](int i) {
      const int row = i < entries ? s_row[i] : -1;
      return row >= 0 ? *reinterpret_cast<const float2*>(c.scale + 2 * (int64_t)(row >> (c.blog2 + 1)))
                      : make_float2(0.0f, 0.0f);
    };
    for (int i = kWave + lane; i < entries; i += kWave) s_sc[i] = scales(i);
    const float2 sc0 = scales(lane);
    Chunk x[PF];
#pragma unroll
    for (int j = 0; j < PF; ++j) fetch(first + j * stride, x[j]);
    if (lane < entries) s_sc[lane] = sc0;
    tail();
    wave_sync();
    for (int c0 = first; c0 < nchunks; c0 += PF * stride) {
#pragma unroll
      for (int j = 0; j < PF; ++j) {
        const int ci = c0 + j * stride;
        if (ci < nchunks) consume(x[j]);
        fetch(ci + PF * stride, x[j]);
      }
    }
  }

  // bring the row groups to the wavefront's maximum and add them
  rescale(max64(m));
  const float L = sum64(lane % LPR == 0 ? l : 0.0f);
  float sums[4];
  sum_rows<LPR>(acc, sums);
  const bool holds = (lane & 15) < LPR;          // this lane's sums are elements de .. de + 3 of the row
  const int de = ds + 8 * (lane >> 5) + 4 * ((lane >> 4) & 1);
  const float keys = t < 0 ? 0.0f : (float)((nused << c.blog2) + tr + 1 + next);
  T* orow = reinterpret_cast<T*>(p.out) + b * p.osb + h * p.osh + n * p.osn;
  if constexpr (!SPLIT) {
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    if (holds) {
#pragma unroll
      for (int i = 0; i < 4; ++i) orow[de + i] = page_value<T>(sums[i] * inv);
    }
    if (lane == 0) {
      if (p.lse) p.lse[qi] = L != 0.0f ? m + __logf(L) : kNegBig;
      if (p.keys) p.keys[qi] = keys;
    }
    return;
  }
  // the four wavefronts' partials through LDS (past the lists, so no wavefront's list is overwritten)
  float* red = smem_f + kWaves * list8_ints(cap);   // [4][D + 2]
  if (holds) {
#pragma unroll
    for (int i = 0; i < 4; ++i) red[w * (D + 2) + 2 + de + i] = sums[i];
  }
  if (lane == 0) {
    red[w * (D + 2)] = m;
    red[w * (D + 2) + 1] = L;
  }
  __syncthreads();
  if (w != 0) return;
  float M = kLowest, Lt = 0.0f, f[kWaves];
#pragma unroll
  for (int s = 0; s < kWaves; ++s)
    if (red[s * (D + 2) + 1] != 0.0f) M = fmaxf(M, red[s * (D + 2)]);
#pragma unroll
  for (int s = 0; s < kWaves; ++s) {
    const float Ls = red[s * (D + 2) + 1];
    f[s] = Ls != 0.0f ? __expf(red[s * (D + 2)] - M) : 0.0f;
    Lt += Ls * f[s];
  }
  auto merged = [&](int d) {
    float a = 0.0f;
#pragma unroll
    for (int s = 0; s < kWaves; ++s) a += red[s * (D + 2) + 2 + d] * f[s];
    return a;
  };
  if (p.gsplit == 1) {
    const float inv = Lt != 0.0f ? 1.0f / Lt : 0.0f;
    for (int d = lane; d < D; d += kWave) orow[d] = page_value<T>(merged(d) * inv);
    if (lane == 0) {
      if (p.lse) p.lse[qi] = Lt != 0.0f ? M + __logf(Lt) : kNegBig;
      if (p.keys) p.keys[qi] = keys;
    }
    return;
  }
  // several workgroups: each writes its partial through to memory and counts itself in; the last to arrive joins them
  // and resets the counter (no workgroup waits for another)
  float* part = p.ws + (qi * p.gsplit + g) * (D + 2);
  for (int d = lane; d < D; d += kWave) stgf_dc(part + 2 + d, merged(d));
  if (lane == 0) {
    stgf_dc(part, M);
    stgf_dc(part + 1, Lt);
    if (g == 0 && p.keys) p.keys[qi] = keys;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the partial has reached memory
  int last = 0;
  if (lane == 0)
    last = __hip_atomic_fetch_add(p.cnt + qi, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           (uint32_t)(p.gsplit - 1);
  if (!__shfl(last, 0, kWave)) return;
  const float* base = p.ws + qi * p.gsplit * (D + 2);
  float ms = kLowest, Ls = 0.0f;
  if (lane < p.gsplit) {
    ms = ldgf_dc(base + lane * (D + 2));
    Ls = ldgf_dc(base + lane * (D + 2) + 1);
  }
  const float Mq = max64(Ls != 0.0f ? ms : kLowest);
  const float fac = Ls != 0.0f ? __expf(ms - Mq) : 0.0f;
  const float Lq = sum64(Ls * fac);
  const float inv = Lq != 0.0f ? 1.0f / Lq : 0.0f;
  float* s_fac = red;   // this wavefront has read its partials
  wave_sync();
  s_fac[lane] = fac;
  wave_sync();
  for (int d = lane; d < D; d += kWave) {
    float a = 0.0f;
    for (int s0 = 0; s0 < p.gsplit; s0 += 8) {
      float pv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = s0 + i < p.gsplit ? ldgf_dc(base + (s0 + i) * (D + 2) + 2 + d) : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < p.gsplit) a += pv[i] * s_fac[s0 + i];
    }
    orow[d] = page_value<T>(a * inv);
  }
  if (lane == 0) {
    if (p.lse) p.lse[qi] = Lq != 0.0f ? Mq + __logf(Lq) : kNegBig;
    __hip_atomic_store(p.cnt + qi, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // ready for the next call
  }
}

template <typename T, int D>
int launch8(const Attn8& p, int B, bool split, hipStream_t st) {
  const int cap = list8_cap(p.wl, p.nb_S);
  size_t lds = (size_t)kWaves * list8_ints(cap) * 4;
  const dim3 blk(kWaves * kWave);
  if (split) {
    lds += (size_t)kWaves * (D + 2) * 4;
    hipLaunchKernelGGL((attn8_kernel<T, D, true>), dim3((unsigned)((int64_t)p.Nq * p.gsplit), B * p.H), blk, lds, st, p);
  } else {
    hipLaunchKernelGGL((attn8_kernel<T, D, false>), dim3((unsigned)((p.Nq + kWaves - 1) / kWaves), B * p.H), blk, lds,
                       st, p);
  }
  return check_launch("attn8_kernel");
}

template <typename T>
int dispatch8(const Attn8& p, int B, int D, bool split, hipStream_t st) {
  switch (D) {
    case 16: return launch8<T, 16>(p, B, split, st);
    case 32: return launch8<T, 32>(p, B, split, st);
    case 64: return launch8<T, 64>(p, B, split, st);
    default: return launch8<T, 128>(p, B, split, st);
  }
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_seg_attn8_fwd(const void* q, int dtype, int64_t qsb, int64_t qsh, int64_t qsn, const ta_kv8* cache,
                                int B, int H, int Nq, int D, const int32_t* tq, int64_t tq_sb, const int32_t* ids,
                                const uint8_t* vld, const int32_t* n_tree, int wl, int local, float scale,
                                const int32_t* nb_id, const uint8_t* nb_ok, int nb_S, void* out, int64_t osb,
                                int64_t osh, int64_t osn, float* lse, float* keys, int nsplit, float* ws,
                                int64_t ws_bytes, void* stream) {
  Attn8 p{};
  const int rc = kv8_view(cache, dtype, B, H, D, "ta_seg_attn8_fwd", p.c);
  if (rc != TA_OK) return rc;
  if (Nq < 0 || wl < 0 || wl > 512 || nsplit < 1 || (nsplit > 1 && nsplit % kWaves) || nsplit > kWaves * kWave) {
    set_error("ta_seg_attn8_fwd: bad sizes (at most 512 leaves; nsplit 1 or a multiple of 4, at most 256)");
    return TA_ERR_ARG;
  }
  if (nb_S < 0 || nb_S > kWave || (nb_S > 0 && (nb_id == nullptr || nb_ok == nullptr))) {
    set_error("ta_seg_attn8_fwd: neighbour slots must number at most 64, with ids and flags");
    return TA_ERR_ARG;
  }
  const int Lw = local > 3 ? local : 3;
  if (Lw + 1 > 32) {
    set_error("ta_seg_attn8_fwd: local window must be < 32");
    return TA_ERR_UNSUPPORTED;
  }
  // rows of all pages are addressed by one int32, and a workgroup's grid by 16 bits of (sequence, head)
  if ((p.c.npages << (p.c.blog2 + 1)) > 0x7fffffffLL || (int64_t)B * H > 65535 ||
      (int64_t)Nq * nsplit > 0x7fffffffLL || (int64_t)(wl + nb_S + 1) << p.c.blog2 > 0x3fffffffLL) {
    set_error("ta_seg_attn8_fwd: too large (fewer than 2^31 rows in all pages, at most 65535 (sequence, head) pairs)");
    return TA_ERR_UNSUPPORTED;
  }
  if (Nq == 0) return TA_OK;
  const int sz = dtype == TA_F32 ? 4 : 2;
  if (q == nullptr || out == nullptr || tq == nullptr || (wl > 0 && (ids == nullptr || vld == nullptr))) {
    set_error("ta_seg_attn8_fwd: a missing pointer");
    return TA_ERR_ARG;
  }
  if ((uintptr_t)q % 16 || (qsb * sz) % 16 || (qsh * sz) % 16 || (qsn * sz) % 16) {
    set_error("ta_seg_attn8_fwd: q rows not 16-byte aligned");
    return TA_ERR_ARG;
  }
  const int64_t need = ta_seg_attn_workspace_size(B, H, Nq, D, nsplit);
  if (need > 0 && (ws == nullptr || ws_bytes < need || (uintptr_t)ws % 256)) {
    set_error("ta_seg_attn8_fwd: workspace missing, too small or not 256-byte aligned");
    return TA_ERR_WORKSPACE;
  }
  p.q = q; p.qsb = qsb; p.qsh = qsh; p.qsn = qsn;
  p.H = H; p.Nq = Nq;
  p.tq = tq; p.tq_sb = tq_sb;
  p.ids = ids; p.vld = vld; p.n_tree = n_tree; p.wl = wl;
  p.Lw = Lw;
  p.scale = scale;
  p.gsplit = nsplit > 1 ? nsplit / kWaves : 1;
  p.out = out; p.osb = osb; p.osh = osh; p.osn = osn;
  p.lse = lse; p.keys = keys;
  if (need > 0) {
    p.cnt = reinterpret_cast<uint32_t*>(ws);
    p.ws = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + attn_counter_bytes(B, H, Nq));
  }
  p.nb_id = nb_id; p.nb_ok = nb_ok; p.nb_S = nb_S;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case TA_F32: return dispatch8<float>(p, B, D, nsplit > 1, st);
    case TA_F16: return dispatch8<f16_t>(p, B, D, nsplit > 1, st);
    default: return dispatch8<bf16_t>(p, B, D, nsplit > 1, st);
  }
}
