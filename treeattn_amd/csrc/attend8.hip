// Sparse softmax attention over a cache of 8-bit pages (kv8.hpp): the selected leaf blocks, the own block and the
// static keys of each query, as attend.hip has it over caches in the model's type.
//
// For key j of a page with scales (sk, sv), k_j = sk * k8_j and v_j = sv * v8_j:
//   s_j = scale * sk * (q . k8_j),  out = sum_j e^(s_j - M) sv * v8_j / sum_j e^(s_j - M)
// so a page's scales cost one multiplication per key, not per element.  Keys of the block that the tail holds are read
// from there, unrounded.  Sums, maxima and the accumulators are float32; the output is rounded once.
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

  float qv[E];
  load_row_g<T, E>(reinterpret_cast<const T*>(p.q) + b * p.qsb + h * p.qsh + n * p.qsn + ds, qv);
  int t = p.tq[b * p.tq_sb + n];
  if (t < 0 || t >= c.tcap) t = -1;   // out of range: attend nothing
  const int held = c.tail_block[b * c.tb_sb + h];
  const int32_t* idr = p.ids + qi * p.wl;
  const uint8_t* vr = p.vld + qi * p.wl;
  const int32_t* trow = c.table + b * c.sb + h * c.sh;
  int nv = 0;
  for (int i0 = 0; i0 < p.wl; i0 += kWave) {
    const int i = i0 + lane;
    nv += __popcll(__ballot(i < p.wl && vr[i] != 0));
  }
  const int nt = p.n_tree ? p.n_tree[qi] : p.wl;
  int nused = t < 0 ? 0 : (nv < nt ? nv : (nt > 0 ? nt : 0));
  const int own = t < 0 ? -1 : t >> c.blog2;
  const int lb = t < 0 ? 0 : own << c.blog2;

  // An entry: block id, its page's first row and scales; row -1 where the block has no page, lies outside the table or
  // is the one in the tail (whose keys are added from there).
  auto entry = [&](int slot, int id, int row_in) {
    int row = -1;
    float2 sc = make_float2(1.0f, 1.0f);
    if (id >= 0 && id < nblk && id != held) {
      const int pg = c.page(trow, id);
      if (pg >= 0) {
        row = (pg << (c.blog2 + 1)) + row_in;
        sc = *reinterpret_cast<const float2*>(c.scale + 2 * (int64_t)pg);
      }
    }
    s_row[slot] = row;
    s_id[slot] = id;
    s_sc[slot] = sc;
  };
  bool all = false;   // the tail's block is among the selected ones
  for (int i0 = 0; i0 < nused; i0 += kWave) {
    const int i = i0 + lane;
    const int id = i < nused ? idr[i] : -1;
    if (i < nused) entry(i, id, 0);
    all |= __ballot(i < nused && id == held && id >= 0) != 0;
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
    if (keep) entry(nused + __popcll(km & ((1ull << lane) - 1)), id, 0);
    all |= __ballot(keep && id == held) != 0;
    nused += __popcll(km);
    wave_sync();
  }
  // static keys [0, t, t-1, ..., t-Lw+1]: those >= 0, outside the own block, whose block is not used, the sink once
  int pe = -1;
  if (lane <= p.Lw && t >= 0) pe = lane == 0 ? 0 : t - (lane - 1);
  bool keep = pe >= 0 && pe < lb && !(lane > 0 && pe == 0);
  if (keep) {
    const int lf = pe >> c.blog2;
    for (int i = 0; i < nused; ++i)
      if (s_id[i] == lf) keep = false;
  }
  const uint64_t bal = __ballot(keep);
  const int next = __popcll(bal);
  const int nblocks = nused + (t < 0 ? 0 : 1);   // the own block is the last of the blocks
  if (keep) entry(nblocks + __popcll(bal & ((1ull << lane) - 1)), pe >> c.blog2, pe & mask);
  if (t >= 0 && lane == 0) entry(nused, own, 0);
  wave_sync();
  const int nl = nblocks << c.blog2;    // keys of the blocks (the own block's past t masked), then the static ones
  const int N8 = nl + next;

  const char* kb = reinterpret_cast<const char*>(c.pool) + ds;
  const int64_t vofs = (int64_t)leaf * D;
  const int nchunks = (N8 + KPC - 1) / KPC;
  const int stride = SPLIT ? p.gsplit * kWaves : 1;
  const int first = SPLIT ? g * kWaves + w : 0;
  const int tr = t & mask;

  struct Chunk {
    uint4 k[NL], v[NL];
    float ks[NL], vs[NL];
    bool ok[NL];
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
      int r0 = -1;
      float2 sc = make_float2(0.0f, 0.0f);
      if (N8 > 0) {
        r0 = s_row[e];
        sc = s_sc[e];
      }
      x.ok[i] = key < N8 && r0 >= 0 && !(blk && e == nused && rr > tr);
      row[i] = x.ok[i] ? r0 + rr : 0;
      x.ks[i] = sc.x * p.scale;
      x.vs[i] = sc.y;
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
    float cm = kLowest;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      sc[i] = group_sum<LPR>(sc[i]) * x.ks[i];
      if (x.ok[i]) cm = fmaxf(cm, sc[i]);
    }
    rescale(fmaxf(m, cm));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const float pw = x.ok[i] ? __expf(sc[i] - m) : 0.0f;
      l += pw;
      const float pv = x.ok[i] ? pw * x.vs[i] : 0.0f;
      float vv[E];
      e4m3_x16(x.v[i], vv);
      if (x.ok[i]) {
#pragma unroll
        for (int d = 0; d < E; ++d) acc[d] = fmaf(pv, vv[d], acc[d]);
      }
    }
  };

  if (nchunks > 0) {
    Chunk x[PF];
#pragma unroll
    for (int j = 0; j < PF; ++j) fetch(first + j * stride, x[j]);
    for (int c0 = first; c0 < nchunks; c0 += PF * stride) {
#pragma unroll
      for (int j = 0; j < PF; ++j) {
        const int ci = c0 + j * stride;
        if (ci < nchunks) consume(x[j]);
        fetch(ci + PF * stride, x[j]);
      }
    }
  }

  // the block in the tail: all its rows when selected, those up to t when it is the own block, else its static keys
  if (t >= 0 && held >= 0 && (held <= own || all)) {
    const bool mine = held == own;
    const T* tk = reinterpret_cast<const T*>(c.tail) + b * c.tail_sb + h * c.tail_sh + ds;
    const int rows = mine ? tr + 1 : leaf;
    for (int r0 = first * RPI; r0 < rows; r0 += stride * RPI) {
      const int r = r0 + rg;
      const int pos = (held << c.blog2) + r;
      const bool ok = r < rows && (mine || all || pos == 0 || pos > t - p.Lw);
      if (__ballot(ok) == 0) continue;
      const int rc = ok ? r : 0;
      float kv[E], vv[E];
      load_row_g<T, E>(tk + (int64_t)rc * D, kv);
      load_row_g<T, E>(tk + (int64_t)leaf * D + (int64_t)rc * D, vv);
      float s = 0.0f;
#pragma unroll
      for (int d = 0; d < E; ++d) s = fmaf(qv[d], kv[d], s);
      s = group_sum<LPR>(s) * p.scale;
      rescale(fmaxf(m, ok ? s : kLowest));
      if (ok) {
        const float pw = __expf(s - m);
        l += pw;
#pragma unroll
        for (int d = 0; d < E; ++d) acc[d] = fmaf(pw, vv[d], acc[d]);
      }
    }
  }

  // bring the row groups to the wavefront's maximum and add them
  {
    const float M = wave_max(m);
    rescale(M);
  }
  float L = wave_sum(lane % LPR == 0 ? l : 0.0f);
#pragma unroll
  for (int o = LPR; o < kWave; o <<= 1) {
#pragma unroll
    for (int d = 0; d < E; ++d) acc[d] += __shfl_xor(acc[d], o, kWave);
  }
  const float keys = t < 0 ? 0.0f : (float)((nused << c.blog2) + tr + 1 + next);
  T* orow = reinterpret_cast<T*>(p.out) + b * p.osb + h * p.osh + n * p.osn;
  if constexpr (!SPLIT) {
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    if (rg == 0) {
#pragma unroll
      for (int d = 0; d < E; ++d) orow[ds + d] = from_f32<T>(acc[d] * inv);
    }
    if (lane == 0) {
      if (p.lse) p.lse[qi] = L != 0.0f ? m + __logf(L) : kNegBig;
      if (p.keys) p.keys[qi] = keys;
    }
    return;
  }
  // the four wavefronts' partials through LDS (past the lists, so no wavefront's list is overwritten)
  float* red = smem_f + kWaves * list8_ints(cap);   // [4][D + 2]
  if (rg == 0) {
#pragma unroll
    for (int d = 0; d < E; ++d) red[w * (D + 2) + 2 + ds + d] = acc[d];
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
    for (int d = lane; d < D; d += kWave) orow[d] = from_f32<T>(merged(d) * inv);
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
  const float Mq = wave_max(Ls != 0.0f ? ms : kLowest);
  const float fac = Ls != 0.0f ? __expf(ms - Mq) : 0.0f;
  const float Lq = wave_sum(Ls * fac);
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
    orow[d] = from_f32<T>(a * inv);
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
