// Rows of many tensors copied by one list of (from, to) pairs: the pages of all layers of a forked or moved sequence, the
// scales of 8-bit pages, the rows of a sequence's tree state.
//
// Nothing to compute: bound by bytes, each row read and written once, and for few pairs by launches, so that up to 32
// tensors go in one: a line of the grid each, as long as the longest needs (a search for a workgroup's tensor would be a chain
// of scalar loads in front of its first byte).  A workgroup takes a piece of kPiece bytes of one row, or as many whole rows as
// fit such a piece.  A pair with an id outside its tensor copies nothing.
//
// Loads and stores that the caches need not keep: what the stores leave in the second caches is written back when the kernel
// ends (in one session 96 pages of 16 KiB in 12 layers 20.5 us so and 8.6 us with nontemporal ones, eight pages of one layer 4.3
// and 2.5; three sets of pools in turns 10.1, 3.7 TB/s).  6143 8-bit pages of 12 layers 228 us, 5.3 TB/s.
//
// The reference keeps one contiguous cache a sequence (engine.py:26-27) and has no counterpart.
#include "common.hpp"

namespace ta {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 32;            // of one launch
constexpr int kUnroll = 4;
constexpr int64_t kPiece = (int64_t)kThreads * kUnroll * 16;

struct RowTensor {
  const char* from;
  char* to;
  int64_t row;          // bytes of a row
  int64_t from_rows, to_rows;
  int64_t pieces;       // workgroups a row, or
  int rows;             // rows a workgroup (pieces == 1)
  unsigned wgs;
  int width;            // bytes of an access: 16, 4 or 1
};
struct CopyArgs {
  RowTensor t[kTensors];
  int n;
  int pairs;
  const int32_t* src;
  const int32_t* dst;
};

template <typename V>
__device__ __forceinline__ void copy_bytes(const char* from, char* to, int64_t bytes) {
  const V* s = reinterpret_cast<const V*>(from);
  V* d = reinterpret_cast<V*>(to);
  const int n = (int)(bytes / (int64_t)sizeof(V));
  for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * kUnroll) {
    V v[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (i0 + j * kThreads < n) v[j] = __builtin_nontemporal_load(s + i0 + j * kThreads);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (i0 + j * kThreads < n) __builtin_nontemporal_store(v[j], d + i0 + j * kThreads);
  }
}

template <typename V>
__device__ __forceinline__ void copy_small(const CopyArgs& p, const RowTensor& t, int64_t pair0) {
  const int per = (int)(t.row / (int64_t)sizeof(V));   // accesses a row
  const int all = t.rows * per;
  for (int i = threadIdx.x; i < all; i += kThreads) {
    const int64_t pair = pair0 + i / per;
    if (pair >= p.pairs) break;
    const int64_t a = p.src[pair], b = p.dst[pair];
    if (a < 0 || a >= t.from_rows || b < 0 || b >= t.to_rows) continue;
    const int64_t o = (int64_t)(i % per) * (int64_t)sizeof(V);
    __builtin_nontemporal_store(__builtin_nontemporal_load(reinterpret_cast<const V*>(t.from + a * t.row + o)),
                                reinterpret_cast<V*>(t.to + b * t.row + o));
  }
}

__global__ __launch_bounds__(kThreads) void copy_rows_kernel(CopyArgs p) {
  const RowTensor t = p.t[blockIdx.y];
  const unsigned at = blockIdx.x;
  if (at >= t.wgs) return;
  if (t.rows > 0) {
    const int64_t pair0 = (int64_t)at * t.rows;
    if (t.width == 16) copy_small<u32x4_t>(p, t, pair0);
    else if (t.width == 4) copy_small<uint32_t>(p, t, pair0);
    else copy_small<uint8_t>(p, t, pair0);
    return;
  }
  const unsigned pieces = (unsigned)t.pieces, pair = pieces == 1 ? at : at / pieces;
  const int64_t o = (int64_t)(at - pair * pieces) * kPiece;
  const int64_t a = p.src[pair], b = p.dst[pair];
  if (a < 0 || a >= t.from_rows || b < 0 || b >= t.to_rows) return;
  const int64_t bytes = t.row - o < kPiece ? t.row - o : kPiece;
  const char* from = t.from + a * t.row + o;
  char* to = t.to + b * t.row + o;
  if (t.width == 16) copy_bytes<u32x4_t>(from, to, bytes);
  else if (t.width == 4) copy_bytes<uint32_t>(from, to, bytes);
  else copy_bytes<uint8_t>(from, to, bytes);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_copy_rows(int n, const void* const* from, void* const* to, const int64_t* row_bytes,
                            const int64_t* from_rows, const int64_t* to_rows, const int32_t* src, const int32_t* dst,
                            int pairs, void* stream) {
  if (n < 0 || pairs < 0 || (n > 0 && (from == nullptr || to == nullptr || row_bytes == nullptr || from_rows == nullptr ||
                                       to_rows == nullptr)) ||
      (pairs > 0 && (src == nullptr || dst == nullptr))) {
    set_error("ta_copy_rows: bad sizes or a missing pointer");
    return TA_ERR_ARG;
  }
  for (int i = 0; i < n; ++i)
    if (row_bytes[i] < 0 || row_bytes[i] > ((int64_t)1 << 40) || from_rows[i] < 0 || to_rows[i] < 0 ||
        (row_bytes[i] > 0 && ((from_rows[i] > 0 && from[i] == nullptr) || (to_rows[i] > 0 && to[i] == nullptr)))) {
      set_error("ta_copy_rows: bad sizes or a missing pointer");
      return TA_ERR_ARG;
    }
  if (pairs == 0) return TA_OK;
  CopyArgs p;
  p.pairs = pairs;
  p.src = src;
  p.dst = dst;
  for (int i0 = 0; i0 < n;) {
    unsigned longest = 0;
    p.n = 0;
    for (; i0 < n && p.n < kTensors; ++i0) {
      const int64_t row = row_bytes[i0];
      if (row == 0) continue;
      RowTensor t{(const char*)from[i0], (char*)to[i0], row, from_rows[i0], to_rows[i0], 1, 0, 0, 1};
      const uintptr_t bits = (uintptr_t)from[i0] | (uintptr_t)to[i0] | (uintptr_t)row;
      t.width = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1);
      int64_t wgs;
      if (row * 2 <= kPiece / (16 / t.width)) {
        t.rows = (int)(kPiece / (16 / t.width) / row);
        wgs = (pairs + t.rows - 1) / t.rows;
      } else {
        t.pieces = (row + kPiece - 1) / kPiece;
        wgs = t.pieces * pairs;
      }
      if (wgs > 0x7fffffffLL) {
        set_error("ta_copy_rows: too large");
        return TA_ERR_UNSUPPORTED;
      }
      t.wgs = (unsigned)wgs;
      longest = t.wgs > longest ? t.wgs : longest;
      p.t[p.n++] = t;
    }
    if (p.n == 0) break;
    hipLaunchKernelGGL(copy_rows_kernel, dim3(longest, p.n), dim3(kThreads), 0, (hipStream_t)stream, p);
    const int rc = check_launch("copy_rows_kernel");
    if (rc != TA_OK) return rc;
  }
  return TA_OK;
}
