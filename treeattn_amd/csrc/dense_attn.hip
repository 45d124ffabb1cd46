// Attention of new tokens over a whole decode cache: every key from position 0 to the query's own.
//
//   s_j = scale * (q . k_j),  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse = m + log sum_j e^(s_j - m)
//
// over the keys j = 0 .. t that have a page.  Query head h reads key head h / (Hq / H).  Scores, sums and the accumulators
// are float32, the output is rounded once.
//
// Reference functions replaced: engine.py:74-81 (DenseState.attend).
#include "attn.hpp"

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
};

// A wavefront a query: a lane scores a key, then holds elements lane and lane + 64 of the output.
template <typename T>
__global__ __launch_bounds__(kWave) void dense_attn_kernel(Dense p) {
  const int lane = lane_id();
  const int n = blockIdx.x, hq = blockIdx.y % p.Hq, b = blockIdx.y / p.Hq;
  const int h = hq / p.G;
  int t = p.tq[b * p.tq_sb + n];
  if (t < 0 || t >= p.Tk) t = -1;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.qsb + hq * p.qsh + n * p.qsn;
  const T* kb = reinterpret_cast<const T*>(p.k) + (p.ptab ? 0 : b * p.ksb + h * p.ksh);
  const T* vb = reinterpret_cast<const T*>(p.v) + (p.ptab ? 0 : b * p.vsb + h * p.vsh);
  float m = kLowest, l = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int j0 = 0; j0 <= t; j0 += kWave) {
    const int j = j0 + lane;
    int64_t ko = -1, vo = -1;
    if (j <= t) {
      if (p.ptab) {
        const int pg = p.ptab[b * p.pt_sb + h * p.pt_sh + (j >> p.blog2)];
        const int r = j & ((1 << p.blog2) - 1);
        if (pg >= 0 && pg < p.npages) {
          ko = pg * p.pstride + r * p.kst;
          vo = pg * p.pstride + r * p.vst;
        }
      } else {
        ko = j * p.kst;
        vo = j * p.vst;
      }
    }
    float s = 0.0f;
    if (ko >= 0)
      for (int d = 0; d < p.D; ++d) s = fmaf(to_f32(q[d]), to_f32(kb[ko + d]), s);
    s *= p.scale;
    const float mn = fmaxf(m, wave_max(ko >= 0 ? s : kLowest));
    const float alpha = __expf(m - mn);
    m = mn;
    const float w = ko >= 0 ? __expf(s - m) : 0.0f;
    l = l * alpha + wave_sum(w);
    acc[0] *= alpha;
    acc[1] *= alpha;
    for (int i = 0; i < kWave; ++i) {
      const int64_t o = __shfl(vo, i, kWave);
      const float wi = __shfl(w, i, kWave);
      if (o < 0) continue;
      if (lane < p.D) acc[0] = fmaf(wi, to_f32(vb[o + lane]), acc[0]);
      if (lane + kWave < p.D) acc[1] = fmaf(wi, to_f32(vb[o + lane + kWave]), acc[1]);
    }
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  T* o = reinterpret_cast<T*>(p.out) + b * p.osb + hq * p.osh + n * p.osn;
  if (lane < p.D) o[lane] = from_f32<T>(acc[0] * inv);
  if (lane + kWave < p.D) o[lane + kWave] = from_f32<T>(acc[1] * inv);
  if (lane == 0 && p.lse) p.lse[((int64_t)b * p.Hq + hq) * p.Nq + n] = l != 0.0f ? m + __logf(l) : kNegBig;
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int64_t ta_dense_attn_workspace_size(int B, int Hq, int H, int Nq, int D, int nsplit) {
  if (B <= 0 || H <= 0 || Hq <= 0 || Nq <= 0 || nsplit <= 4) return 0;
  const int64_t tiles = (int64_t)B * H * (((int64_t)(Hq / H) * Nq + 15) / 16);
  return (tiles * 4 + 255) / 256 * 256 + tiles * (nsplit / 4) * 16 * (D + 2) * 4;
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
  if (B < 0 || H < 1 || Hq < 1 || Hq % H || Nq < 0 || Tk < 1 || (int64_t)B * Hq > 65535) {
    set_error("ta_dense_attn_fwd: bad sizes (query heads a multiple of the key heads, at most 65535 (sequence, head) pairs)");
    return TA_ERR_ARG;
  }
  if (nsplit < 1 || (nsplit > 1 && nsplit % 4) || nsplit > 1024) {
    set_error("ta_dense_attn_fwd: nsplit must be 1 or a multiple of 4, at most 1024");
    return TA_ERR_ARG;
  }
  if (pages && (pages->table == nullptr || pages->num_pages <= 0 || pages->block_log2 < 0 || pages->block_log2 > 14)) {
    set_error("ta_dense_attn_fwd: bad page description");
    return TA_ERR_ARG;
  }
  if (B == 0 || Nq == 0) return TA_OK;
  if (q == nullptr || k == nullptr || v == nullptr || tq == nullptr || out == nullptr) {
    set_error("ta_dense_attn_fwd: a missing pointer");
    return TA_ERR_ARG;
  }
  const int sz = dtype == TA_F32 ? 4 : 2;
  const int64_t bits = (int64_t)((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) | (qsb | qsh | qsn | kst | vst) * sz |
                       (pages ? pages->page_stride * sz : (ksb | ksh | vsb | vsh) * sz);
  if (bits % 16) {
    set_error("ta_dense_attn_fwd: q, K and V rows must be 16-byte aligned");
    return TA_ERR_ARG;
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
  const dim3 grid(Nq, B * Hq), blk(kWave);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TA_F32) hipLaunchKernelGGL((dense_attn_kernel<float>), grid, blk, 0, st, p);
  else if (dtype == TA_F16) hipLaunchKernelGGL((dense_attn_kernel<f16_t>), grid, blk, 0, st, p);
  else hipLaunchKernelGGL((dense_attn_kernel<bf16_t>), grid, blk, 0, st, p);
  return check_launch("dense_attn_kernel");
}
