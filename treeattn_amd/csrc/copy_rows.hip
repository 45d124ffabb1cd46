// Rows of many tensors copied by one list of (from, to) pairs: the pages of all layers of a forked or moved sequence, the
// scales of 8-bit pages, the rows of a sequence's tree state.
//
// Nothing to compute: bound by bytes, each row read and written once, and for few pairs by launches, so that up to 32
// tensors go in one.  A workgroup takes a piece of kPiece bytes of one row, or as many whole rows of one tensor as fit
// such a piece.  A pair with an id outside its tensor copies nothing.
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
  int64_t first;        // its first workgroup
  int64_t pieces;       // workgroups a row, or
  int rows;             // rows a workgroup (pieces == 1)
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
      if (i0 + j * kThreads < n) v[j] = s[i0 + j * kThreads];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (i0 + j * kThreads < n) d[i0 + j * kThreads] = v[j];
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
    *reinterpret_cast<V*>(t.to + b * t.row + o) = *reinterpret_cast<const V*>(t.from + a * t.row + o);
  }
}

__global__ __launch_bounds__(kThreads) void copy_rows_kernel(CopyArgs p) {
  const int64_t wg = blockIdx.x;
  int k = 0;
  while (k + 1 < p.n && p.t[k + 1].first <= wg) ++k;
  const RowTensor t = p.t[k];
  const int64_t at = wg - t.first;
  if (t.rows > 0) {
    const int64_t pair0 = at * t.rows;
    if (t.width == 16) copy_small<uint4>(p, t, pair0);
    else if (t.width == 4) copy_small<uint32_t>(p, t, pair0);
    else copy_small<uint8_t>(p, t, pair0);
    return;
  }
  const int64_t pair = at / t.pieces, o = (at % t.pieces) * kPiece;
  const int64_t a = p.src[pair], b = p.dst[pair];
  if (a < 0 || a >= t.from_rows || b < 0 || b >= t.to_rows) return;
  const int64_t bytes = t.row - o < kPiece ? t.row - o : kPiece;
  const char* from = t.from + a * t.row + o;
  char* to = t.to + b * t.row + o;
  if (t.width == 16) copy_bytes<uint4>(from, to, bytes);
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
    int64_t blocks = 0;
    p.n = 0;
    while (i0 < n && p.n < kTensors) {
      const int64_t row = row_bytes[i0];
      RowTensor t{(const char*)from[i0], (char*)to[i0], row, from_rows[i0], to_rows[i0], blocks, 1, 0, 1};
      const uintptr_t bits = (uintptr_t)from[i0] | (uintptr_t)to[i0] | (uintptr_t)row;
      t.width = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1);
      int64_t add = 0;
      if (row > 0 && row * 2 <= kPiece / (16 / t.width)) {
        t.rows = (int)(kPiece / (16 / t.width) / row);
        add = (pairs + t.rows - 1) / t.rows;
      } else if (row > 0) {
        t.pieces = (row + kPiece - 1) / kPiece;
        add = t.pieces * pairs;
      }
      if (add > 0x7fffffffLL) {
        set_error("ta_copy_rows: too large");
        return TA_ERR_UNSUPPORTED;
      }
      if (blocks + add > 0x7fffffffLL) break;   // the rest in a launch of its own
      if (add > 0) {
        p.t[p.n++] = t;
        blocks += add;
      }
      ++i0;
    }
    if (blocks == 0) continue;
    hipLaunchKernelGGL(copy_rows_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, p);
    const int rc = check_launch("copy_rows_kernel");
    if (rc != TA_OK) return rc;
  }
  return TA_OK;
}
