// Writing a decode cache of 8-bit pages: the append of one decoded token and the fill from a prompt.
//
// The reference keeps the cache in the model's type (engine.py:26-27, 41-55 SegState.add, 57-71 fill); here a leaf
// block is rounded to e4m3 once, when its last row has arrived, with one scale for its keys and one for its values.
// Until then its rows stand unrounded in the sequence's tail, so the scale is that of the whole block, a prompt and
// the same tokens one by one give the same bytes, and the node sums are those of the unrounded keys.  Scales are
// powers of two: e4m3 has the same relative step over its whole range, so a scale that is up to twice too large
// costs nothing but the lowest of its subnormals, and multiplying by it is exact.
#include "kv8.hpp"

namespace ta {

int kv8_view(const ta_kv8* c, int dtype, int B, int H, int D, const char* who, Kv8& out) {
  const int sz = dtype == TA_F32 ? 4 : 2;
  if (dtype != TA_F32 && dtype != TA_F16 && dtype != TA_BF16) {
    set_error(std::string(who) + ": unknown dtype");
    return TA_ERR_ARG;
  }
  if (D != 16 && D != 32 && D != 64 && D != 128) {
    set_error(std::string(who) + ": head dim must be 16, 32, 64 or 128");
    return TA_ERR_UNSUPPORTED;
  }
  if (c == nullptr || c->pool == nullptr || c->scale == nullptr || c->table == nullptr || c->tail == nullptr ||
      c->tail_block == nullptr || c->num_pages <= 0 || c->num_pages > 0x7fffffffLL || c->block_log2 < 1 ||
      c->block_log2 > 14 || c->tcap <= 0 || B <= 0 || H <= 0) {
    set_error(std::string(who) + ": bad cache description (pool, scale, table, tail and tail_block, 1 to 2^31 - 1 "
                                 "pages of 2 to 16384 rows)");
    return TA_ERR_ARG;
  }
  if (((uintptr_t)c->pool | (uintptr_t)c->tail) % 16 || (uintptr_t)c->scale % 8 || (c->tail_sb * sz) % 16 ||
      (c->tail_sh * sz) % 16 || (uintptr_t)c->table % 4 || (uintptr_t)c->tail_block % 4) {
    set_error(std::string(who) + ": the pages and the tail must be 16-byte aligned, the scales 8-byte aligned");
    return TA_ERR_ARG;
  }
  out = Kv8{(uint8_t*)c->pool, c->scale,  c->table,   c->sb,         c->sh, c->num_pages,  c->tail,
            c->tail_sb,        c->tail_sh, c->tail_block, c->tb_sb, c->block_log2, c->tcap};
  return TA_OK;
}

namespace {

constexpr int kAppendThreads = 256;

struct LevelRW8 {
  float* ptr[kMaxLevels];
  int64_t sb[kMaxLevels];
  int64_t sh[kMaxLevels];
};

// VE elements of T (16 bytes) -> floats
template <typename T> constexpr int vec_elems() { return 16 / (int)sizeof(T); }

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[vec_elems<T>()]) {
  load_row_g<T, vec_elems<T>()>(p, f);
}

// One 16-byte vector of T, rounded with exponent e, stored at byte address dst (VE bytes).
template <typename T>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&f)[vec_elems<T>()], int e) {
  if constexpr (vec_elems<T>() == 8) {
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(e4m3_x4(f[0], f[1], f[2], f[3], e), e4m3_x4(f[4], f[5], f[6], f[7], e));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = e4m3_x4(f[0], f[1], f[2], f[3], e);
  }
}

// One workgroup per (sequence, head).  A row is 2 D values, so what a call costs is a launch and its round trips (position,
// page, tag, then the rows): 32 x 12 rows of 64 bf16 3.6 us.  The call that ends a block reads it once more from L2: its
// sums by runs of rows beside the rounding, 6 blocks of 32 x 64 float32 6.5 us (8.8 with the sums by one thread a
// dimension and a second read for the rounding).
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void kv8_append_kernel(Kv8 c, const T* __restrict__ kn,
                                                                    const T* __restrict__ vn, int64_t nsb, int64_t nsh,
                                                                    int64_t vnsb, int64_t vnsh, int H, int D,
                                                                    const int32_t* __restrict__ t_pos, LevelRW8 lv,
                                                                    int n_levels, int arity_log2) {
  extern __shared__ float stk[];   // carry stacks [16][threads]
  __shared__ float s_max[2][kAppendThreads / kWave];
  constexpr int VE = vec_elems<T>();
  const int tid = threadIdx.x;
  const int b = blockIdx.x / H, h = blockIdx.x % H;
  const int t = t_pos[b];
  if (t < 0 || t >= c.tcap) return;
  const int leaf = 1 << c.blog2;
  const int blk = t >> c.blog2, r = t & (leaf - 1);
  const int pg = c.page(c.table + b * c.sb + h * c.sh, blk);
  if (pg < 0) return;   // no page for the block: nothing stored, no node formed
  T* tk = reinterpret_cast<T*>(c.tail) + b * c.tail_sb + h * c.tail_sh;
  const int64_t half = (int64_t)leaf * D;
  T* tv = tk + half;
  uint8_t* page = c.pool + (int64_t)pg * 2 * half;
  int32_t* tag = c.tail_block + b * c.tb_sb + h;
  const int held = *tag;
  if (held != blk && r > 0) {
    // the tail holds another block (the caller went back to an earlier position): this block's rows before t come
    // back from its page
    const float ks = c.scale[2 * (int64_t)pg], vs = c.scale[2 * (int64_t)pg + 1];
    for (int64_t i = (int64_t)tid * 16; i < (int64_t)r * D; i += kAppendThreads * 16) {
      float f[16];
      e4m3_x16(ldg16(page + i), f);
#pragma unroll
      for (int u = 0; u < 16; ++u) tk[i + u] = page_value<T>(f[u] * ks);
      e4m3_x16(ldg16(page + half + i), f);
#pragma unroll
      for (int u = 0; u < 16; ++u) tv[i + u] = page_value<T>(f[u] * vs);
    }
  }
  if (tid < 2 * D) {
    const bool isv = tid >= D;
    const int d = isv ? tid - D : tid;
    const T x = isv ? vn[b * vnsb + h * vnsh + d] : kn[b * nsb + h * nsh + d];
    (isv ? tv : tk)[(int64_t)r * D + d] = x;
  }
  __syncthreads();   // every thread has read the tag, the tail's rows are written
  if (tid == 0) *tag = blk;
  if (r != leaf - 1) return;

  // The block is whole.  Its nodes' first level: thread (segment, d) sums an aligned run of rows of dimension d by adjacent
  // pairs, and the runs are joined the same way -- the tree of sums ta_level_sums forms, so the same bits.  The loads of the
  // runs and of the whole block are in flight together.
  const int S = n_levels > 0 ? (kAppendThreads / D < leaf / 2 ? kAppendThreads / D : leaf / 2) : 0;   // runs
  const int seg = tid / D, d = tid % D, run = S > 0 ? leaf / S : 0;
  constexpr int U = 8;
  float rv[U];
  const bool sums = seg < S;
  auto load_run = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r1 = seg * run + i0 + u;
      rv[u] = i0 + u < run ? to_f32(tk[(int64_t)r1 * D + d]) : 0.0f;
    }
  };
  if (sums) load_run(0);
  const int64_t nv = half / VE;
  constexpr int R = 4;                          // vectors of K and of V a thread holds; larger blocks are read twice
  float f[R][VE], g[R][VE];
  float m[2] = {0.0f, 0.0f};
  auto amax = [&](const float (&x)[VE], const float (&y)[VE]) {
#pragma unroll
    for (int u = 0; u < VE; ++u) {
      m[0] = fmaxf(m[0], finite_abs(x[u]));
      m[1] = fmaxf(m[1], finite_abs(y[u]));
    }
  };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t v = (int64_t)i * kAppendThreads + tid;
    if (v < nv) {
      load_vec<T>(tk + v * VE, f[i]);
      load_vec<T>(tv + v * VE, g[i]);
    }
  }
  // run sums: a carry stack of the widths 1, 2, 4, ... below the run's length
  float x = 0.0f;
  if (sums) {
    for (int i0 = 0; i0 < run; i0 += U) {
      if (i0 > 0) load_run(i0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u;
        if (i >= run) break;
        x = (blk == 0 && seg == 0 && i == 0) ? 0.0f : rv[u];   // position 0 counts as zero
        int lvl = 0;
        while ((i >> lvl) & 1) {
          x = __fadd_rn(stk[lvl * kAppendThreads + tid], x);
          ++lvl;
        }
        stk[lvl * kAppendThreads + tid] = x;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if ((int64_t)i * kAppendThreads + tid < nv) amax(f[i], g[i]);
  for (int64_t v = (int64_t)R * kAppendThreads + tid; v < nv; v += kAppendThreads) {
    float y[VE], z[VE];
    load_vec<T>(tk + v * VE, y);
    load_vec<T>(tv + v * VE, z);
    amax(y, z);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    m[s] = wave_max(m[s]);
    if (lane_id() == 0) s_max[s][wave_id()] = m[s];
  }
  __syncthreads();   // the stacks are done with too: a thread's run sum goes to slot tid
  if (sums) stk[tid] = x;
  int e[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float y = s_max[s][0];
#pragma unroll
    for (int w = 1; w < kAppendThreads / kWave; ++w) y = fmaxf(y, s_max[s][w]);
    e[s] = e4m3_exponent(y);
  }
  __syncthreads();
  // nodes: levels j >= 1 that end here need their children before the last, which are read together, eight levels at a time
  if (tid < D && n_levels > 0) {
    for (int w = 1; w < S; w *= 2)
      for (int i = 0; i + w < S; i += 2 * w) stk[i * D + d] = __fadd_rn(stk[i * D + d], stk[(i + w) * D + d]);
    x = stk[d];
    auto level = [&](int j) { return lv.ptr[j] + b * lv.sb[j] + h * lv.sh[j]; };
    level(0)[(int64_t)blk * D + d] = x;
    const int arity = 1 << arity_log2;
    int ends = 1;   // levels whose node ends at t
    while (ends < n_levels && c.blog2 + ends * arity_log2 < 31 &&
           ((t + 1) & ((1 << (c.blog2 + ends * arity_log2)) - 1)) == 0)
      ++ends;
    if (arity == 2) {
      for (int j0 = 1; j0 < ends; j0 += 8) {
        float sib[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          sib[u] = j0 + u < ends ? level(j0 + u - 1)[((int64_t)(t >> (c.blog2 + (j0 + u - 1))) - 1) * D + d] : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (j0 + u >= ends) break;
          x = __fadd_rn(sib[u], x);
          level(j0 + u)[(int64_t)(t >> (c.blog2 + (j0 + u))) * D + d] = x;
        }
      }
    } else {
      for (int j = 1; j < ends; ++j) {
        const int64_t node = t >> (c.blog2 + j * arity_log2);
        const float* child = level(j - 1) + node * arity * D + d;
        float kid[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) kid[k] = k < arity - 1 ? child[(int64_t)k * D] : 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (k == arity - 1) kid[k] = x;
#pragma unroll
        for (int w = 1; w < 16; w *= 2) {
#pragma unroll
          for (int k = 0; k + w < 16; k += 2 * w)
            if (w < arity && k < arity) kid[k] = __fadd_rn(kid[k], kid[k + w]);
        }
        x = kid[0];
        level(j)[node * D + d] = x;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t v = (int64_t)i * kAppendThreads + tid;
    if (v < nv) {
      store_e4m3<T>(page + v * VE, f[i], e[0]);
      store_e4m3<T>(page + half + v * VE, g[i], e[1]);
    }
  }
  for (int64_t v = (int64_t)R * kAppendThreads + tid; v < nv; v += kAppendThreads) {
    float y[VE], z[VE];
    load_vec<T>(tk + v * VE, y);
    load_vec<T>(tv + v * VE, z);
    store_e4m3<T>(page + v * VE, y, e[0]);
    store_e4m3<T>(page + half + v * VE, z, e[1]);
  }
  if (tid < 2) c.scale[2 * (int64_t)pg + tid] = ldexpf(1.0f, e[tid]);
}

// Prompts, bound by the bytes (2 or 4 read, 1 written a value): 8 x 12 prompts of about 7200 rows of 64 bf16, 266 MB, in 56
// us, 4.7 TB/s (a large copy reaches 5.1 to 5.7 here).  A unit is the K or the V rows of one leaf block of one (sequence, head); G lanes (a power of two up to the
// workgroup) serve it, each its R vectors of 16 bytes.  Whole blocks are rounded into their pages, the last partial
// block's rows go to the tail; blocks and rows past a sequence's length are not touched.
template <typename T, int R>
__global__ __launch_bounds__(256) void kv8_fill_kernel(Kv8 c, const T* __restrict__ k, const T* __restrict__ v,
                                                       int64_t ksb, int64_t ksh, int64_t kst, int64_t vsb, int64_t vsh,
                                                       int64_t vst, int H, int T_, int D, int nblk, int64_t units,
                                                       const int32_t* __restrict__ lens, int G) {
  constexpr int VE = vec_elems<T>();
  __shared__ float s_max[4];
  const int tid = threadIdx.x;
  const int64_t unit = blockIdx.x * (int64_t)(256 / G) + tid / G;
  const int g = tid & (G - 1);
  const bool live = unit < units;
  // heads first, then keys and values: neighbours read what lies together in the output of a projection
  const int64_t hs = live ? unit / H : 0;
  const int h = live ? (int)(unit - hs * H) : 0;
  const int side = (int)(hs & 1);
  const int64_t bj = hs >> 1;
  const int b = (int)(bj / nblk), j = (int)(bj - (int64_t)b * nblk);
  const int leaf = 1 << c.blog2;
  const int64_t half = (int64_t)leaf * D;
  int n = T_;
  if (lens != nullptr) n = lens[b];
  n = n < 0 ? 0 : (n < T_ ? n : T_);
  n = n < c.tcap ? n : c.tcap;
  const int rest = n & (leaf - 1);
  const int whole = n >> c.blog2;
  if (live && j == 0 && side == 0 && g == 0 && rest == 0) c.tail_block[b * c.tb_sb + h] = -1;
  int pg = -1;
  if (live && (j < whole || (j == whole && rest > 0))) pg = c.page(c.table + b * c.sb + h * c.sh, j);
  const T* src = side ? v + b * vsb + h * vsh : k + b * ksb + h * ksh;
  const int64_t st = side ? vst : kst;
  const int nrow = pg < 0 ? 0 : (j < whole ? leaf : rest);   // rows of the block that the prompt has
  const int nv = (int)(half / VE);
  const int per = D / VE;                                    // vectors of a row
  auto vec = [&](int i, float (&f)[VE]) {
    const int row = i / per, d = (i % per) * VE;
    load_vec<T>(src + ((int64_t)(j << c.blog2) + row) * st + d, f);
  };
  if (nrow > 0 && nrow < leaf) {   // (a unit's lanes agree; lanes of other units of the wavefront pass by)
    T* dst = reinterpret_cast<T*>(c.tail) + b * c.tail_sb + h * c.tail_sh + side * half;
    for (int i = g; i < nrow * per; i += G) {
      const int row = i / per, d = (i % per) * VE;
      *reinterpret_cast<uint4*>(dst + (int64_t)row * D + d) =
          ldg16(src + ((int64_t)(j << c.blog2) + row) * st + d);
    }
  }
  if (live && j == whole && rest > 0 && side == 0 && g == 0) c.tail_block[b * c.tb_sb + h] = pg < 0 ? -1 : j;
  const bool page = nrow == leaf;
  float x[R > 0 ? R : 1][VE];
  float m = 0.0f;
  if (page) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) vec(i * G + g, x[i]);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int u = 0; u < VE; ++u) m = fmaxf(m, finite_abs(x[i][u]));
    } else {
      for (int i = g; i < nv; i += G) {
        vec(i, x[0]);
#pragma unroll
        for (int u = 0; u < VE; ++u) m = fmaxf(m, finite_abs(x[0][u]));
      }
    }
  }
  for (int o = 1; o < (G < kWave ? G : kWave); o <<= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
  if (G > kWave) {   // uniform over the workgroup; the wavefronts of a unit are consecutive
    if (lane_id() == 0) s_max[wave_id()] = m;
    __syncthreads();
    const int w0 = (tid / G) * (G / kWave);
    for (int w = 0; w < G / kWave; ++w) m = fmaxf(m, s_max[w0 + w]);
  }
  if (!page) return;
  const int e = e4m3_exponent(m);
  uint8_t* dst = c.pool + ((int64_t)pg * 2 + side) * half;
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) store_e4m3<T>(dst + (int64_t)(i * G + g) * VE, x[i], e);
  } else {
    for (int i = g; i < nv; i += G) {
      vec(i, x[0]);
      store_e4m3<T>(dst + (int64_t)i * VE, x[0], e);
    }
  }
  if (g == 0) c.scale[2 * (int64_t)pg + side] = ldexpf(1.0f, e);
}

template <typename T>
int launch_fill(const Kv8& c, const void* k, const void* v, int64_t ksb, int64_t ksh, int64_t kst, int64_t vsb,
                int64_t vsh, int64_t vst, int B, int H, int T_, int D, const int32_t* lens, hipStream_t st) {
  const int64_t nv = ((int64_t)D << c.blog2) / vec_elems<T>();
  // a wavefront a unit as long as eight vectors a lane hold it (64 keys of 64 bf16: 75.7 -> 56.6 us for 8 x 12 x 8191 against four
  // wavefronts with two each), more lanes for larger blocks
  const int G = nv <= 64 ? (int)nv : nv <= 512 ? 64 : nv < 2048 ? (int)(nv / 8) : 256;
  const int64_t R = nv / G;
  const int leaf = 1 << c.blog2;
  const int nblk = T_ > 0 ? (int)(((int64_t)T_ + leaf - 1) / leaf) : 1;
  const int64_t units = (int64_t)B * H * nblk * 2;
  const int64_t grid = (units + 256 / G - 1) / (256 / G);
  if (grid > 0x7fffffffLL) {
    set_error("ta_kv8_fill: too many blocks");
    return TA_ERR_UNSUPPORTED;
  }
#define TA_FILL(RR)                                                                                                  \
  hipLaunchKernelGGL((kv8_fill_kernel<T, RR>), dim3((unsigned)grid), dim3(256), 0, st, c, (const T*)k, (const T*)v, ksb, \
                     ksh, kst, vsb, vsh, vst, H, T_, D, nblk, units, lens, G)
  switch (R) {
    case 1: TA_FILL(1); break;
    case 2: TA_FILL(2); break;
    case 4: TA_FILL(4); break;
    case 8: TA_FILL(8); break;
    default: TA_FILL(0); break;
  }
#undef TA_FILL
  return check_launch("kv8_fill_kernel");
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_kv8_append(const void* k_new, const void* v_new, int dtype, int64_t nsb, int64_t nsh, int64_t vnsb,
                             int64_t vnsh, const ta_kv8* cache, int B, int H, int D, const int32_t* t_pos, int n_levels,
                             float* const* lv_ptr, const int64_t* lv_sb, const int64_t* lv_sh, int arity_log2,
                             void* stream) {
  Kv8 c;
  const int rc = kv8_view(cache, dtype, B, H, D, "ta_kv8_append", c);
  if (rc != TA_OK) return rc;
  if (n_levels < 0 || n_levels > kMaxLevels || arity_log2 < 1 || arity_log2 > 4 || k_new == nullptr ||
      v_new == nullptr || t_pos == nullptr) {
    set_error("ta_kv8_append: bad sizes (at most 32 levels, arity 2 to 16) or a missing pointer");
    return TA_ERR_ARG;
  }
  if (n_levels > 0 && (lv_ptr == nullptr || lv_sb == nullptr || lv_sh == nullptr)) {
    set_error("ta_kv8_append: levels without their addresses or strides");
    return TA_ERR_ARG;
  }
  LevelRW8 lv;
  for (int j = 0; j < n_levels; ++j) {
    if (lv_ptr[j] == nullptr) {
      set_error("ta_kv8_append: levels without their addresses or strides");
      return TA_ERR_ARG;
    }
    lv.ptr[j] = lv_ptr[j];
    lv.sb[j] = lv_sb[j];
    lv.sh[j] = lv_sh[j];
  }
  const size_t lds = (size_t)16 * kAppendThreads * sizeof(float);
#define TA_APPEND(TT)                                                                                             \
  hipLaunchKernelGGL((kv8_append_kernel<TT>), dim3((unsigned)(B * H)), dim3(kAppendThreads), lds, (hipStream_t)stream, c, \
                     (const TT*)k_new, (const TT*)v_new, nsb, nsh, vnsb, vnsh, H, D, t_pos, lv, n_levels, arity_log2)
  switch (dtype) {
    case TA_F32: TA_APPEND(float); break;
    case TA_F16: TA_APPEND(f16_t); break;
    default: TA_APPEND(bf16_t); break;
  }
#undef TA_APPEND
  return check_launch("kv8_append_kernel");
}

extern "C" int ta_kv8_fill(const void* k, const void* v, int dtype, int64_t ksb, int64_t ksh, int64_t kst, int64_t vsb,
                           int64_t vsh, int64_t vst, const ta_kv8* cache, int B, int H, int T, int D,
                           const int32_t* lengths, void* stream) {
  Kv8 c;
  const int rc = kv8_view(cache, dtype, B, H, D, "ta_kv8_fill", c);
  if (rc != TA_OK) return rc;
  const int sz = dtype == TA_F32 ? 4 : 2;
  if (T < 0 || T > c.tcap || (T > 0 && (k == nullptr || v == nullptr))) {
    set_error("ta_kv8_fill: the prompt must have between 0 and tcap positions");
    return TA_ERR_ARG;
  }
  for (int64_t s : {ksb * sz, ksh * sz, kst * sz, vsb * sz, vsh * sz, vst * sz, (int64_t)(uintptr_t)k, (int64_t)(uintptr_t)v})
    if (s % 16) {
      set_error("ta_kv8_fill: k and v rows not 16-byte aligned");
      return TA_ERR_ARG;
    }
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case TA_F32: return launch_fill<float>(c, k, v, ksb, ksh, kst, vsb, vsh, vst, B, H, T, D, lengths, st);
    case TA_F16: return launch_fill<f16_t>(c, k, v, ksb, ksh, kst, vsb, vsh, vst, B, H, T, D, lengths, st);
    default: return launch_fill<bf16_t>(c, k, v, ksb, ksh, kst, vsb, vsh, vst, B, H, T, D, lengths, st);
  }
}
