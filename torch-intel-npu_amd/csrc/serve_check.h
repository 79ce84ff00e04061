// Host-side checks that the entry points of lowbit_decode_hip.h that serve many requests share.
#pragma once
#include <algorithm>
#include <cmath>

#include "../../include/lowbit_decode_hip.h"
#include "abi_util.h"
#include "lb_serve.h"

namespace lb {
namespace abi {

constexpr int64_t kMaxStride = (int64_t)1 << 40, kMaxSeq = (int64_t)1 << 25;   // (launches of up to 2^31 threads)
constexpr size_t kMaxBytes = (size_t)1 << 60;   // (no buffer is larger; sums of a few stay in 64 bits)

// Rows [batch, seq, heads] of dim values of `size` bytes; written ones may not share memory with one another.  pieces: they
// are whole 16-byte pieces.
inline lb_status check_strided(const char *what, const char *name, const lb_rows &v, int64_t batch, int64_t seq, int64_t heads,
                               int64_t dim, size_t size, bool pieces, bool written, Range &range) {
  const size_t align = pieces ? 16 : size;
  if (!v.data || !aligned(v.data, align)) return fail(LB_INVALID_ARGUMENT, "%s: %s must be non-NULL with %zu-byte alignment", what, name, align);
  struct Axis { int64_t size, stride; } axes[3] = {{batch, v.batch_stride}, {seq, v.row_stride}, {heads, v.head_stride}};
  unsigned __int128 span = dim;
  for (Axis &a : axes) {
    if (a.size == 1) a.stride = 0;
    if (a.stride < 0 || a.stride > kMaxStride || (pieces && a.stride * size % 16 != 0))
      return fail(LB_INVALID_ARGUMENT, "%s: strides of %s must be 0 to 2^40 elements%s", what, name, pieces ? " in whole 16-byte pieces" : "");
    span += (unsigned __int128)(a.size - 1) * a.stride;
  }
  if (span > kMaxBytes / 4) return fail(LB_INVALID_ARGUMENT, "%s: %s is past the address space", what, name);
  if (written) {
    std::sort(axes, axes + 3, [](const Axis &a, const Axis &b) { return a.stride < b.stride; });
    int64_t extent = dim;
    for (const Axis &a : axes) {
      if (a.size == 1) continue;
      if (a.stride < extent) return fail(LB_INVALID_ARGUMENT, "%s: rows of %s overlap one another", what, name);
      extent += (a.size - 1) * a.stride;
    }
  }
  range = range_of(v.data, (size_t)span * size, name);
  return range.hi < range.lo ? fail(LB_INVALID_ARGUMENT, "%s: %s does not fit the address space", what, name) : LB_OK;
}

// Whether two sets of checked rows, of the same batch, seq and dim, share no memory: slices of one tensor lie between one another, but
// its outer axes (any of batch, seq and heads, which both step through alike) hold them apart in blocks of `upper` behind `lower`.
inline bool rows_apart(const lb_rows &a, int64_t a_heads, const lb_rows &b, int64_t b_heads, int64_t batch, int64_t seq, int64_t dim, size_t size) {
  const bool swap = reinterpret_cast<uintptr_t>(b.data) < reinterpret_cast<uintptr_t>(a.data);
  const lb_rows &lower = swap ? b : a, &upper = swap ? a : b;
  const size_t bytes = reinterpret_cast<uintptr_t>(upper.data) - reinterpret_cast<uintptr_t>(lower.data);
  struct Axis { int64_t low, up, low_stride, up_stride; };
  const Axis axes[3] = {{batch, batch, lower.batch_stride, upper.batch_stride}, {seq, seq, lower.row_stride, upper.row_stride},
                        {swap ? b_heads : a_heads, swap ? a_heads : b_heads, lower.head_stride, upper.head_stride}};
  for (int outer = 0; outer < 8; ++outer) {
    struct { int64_t size, stride; } steps[3];
    int n = 0;
    int64_t low = dim, up = dim;         // extents of a block's rows
    bool alike = true;
    for (int i = 0; i < 3; ++i) {
      const Axis &x = axes[i];
      if (outer >> i & 1) {
        alike = alike && (x.low == 1 || x.up == 1 || x.low_stride == x.up_stride);
        if (std::max(x.low, x.up) > 1) steps[n++] = {std::max(x.low, x.up), x.low > 1 ? x.low_stride : x.up_stride};
      } else {
        low += x.low == 1 ? 0 : (x.low - 1) * x.low_stride;
        up += x.up == 1 ? 0 : (x.up - 1) * x.up_stride;
      }
    }
    if (!alike || bytes < (size_t)low * size) continue;
    std::sort(steps, steps + n, [](const auto &s, const auto &t) { return s.stride < t.stride; });
    unsigned __int128 extent = bytes + (unsigned __int128)up * size;
    bool apart = true;
    for (int i = 0; i < n; ++i) {
      apart = apart && (unsigned __int128)steps[i].stride * size >= extent;
      extent += (unsigned __int128)(steps[i].size - 1) * steps[i].stride * size;
    }
    if (apart) return true;
  }
  return false;
}

inline lb_status check_array(const char *what, const char *name, const void *p, size_t bytes, size_t align, bool needed, Range &range) {
  range = Range{};
  if (!p && !needed) return LB_OK;
  if (!p || !aligned(p, align)) return fail(LB_INVALID_ARGUMENT, "%s: %s must be non-NULL with %zu-byte alignment", what, name, align);
  range = range_of(p, bytes, name);
  return bytes > kMaxBytes || range.hi < range.lo ? fail(LB_INVALID_ARGUMENT, "%s: %s does not fit the address space", what, name) : LB_OK;
}

inline lb_status check_apart(const char *what, const Range *written, int nw, const Range *read, int nr) {
  for (int i = 0; i < nw; ++i) {
    for (int k = 0; k < nr; ++k)
      if (overlaps(written[i], read[k])) return fail(LB_INVALID_ARGUMENT, "%s: %s overlaps %s", what, written[i].name, read[k].name);
    for (int k = 0; k < i; ++k)
      if (overlaps(written[i], written[k])) return fail(LB_INVALID_ARGUMENT, "%s: %s overlaps %s", what, written[k].name, written[i].name);
  }
  return LB_OK;
}

inline lb_status check_rotation(const char *what, const lb_rotation &r, int64_t head_dim, bool needed, Range &range) {
  if (const lb_status st = check_array(what, "frequencies", r.frequencies, (size_t)r.dims / 2 * 8, 8, needed, range); st != LB_OK) return st;
  if (!r.frequencies) return LB_OK;
  if (r.dims < 2 || r.dims % 2 != 0 || r.dims > head_dim) return fail(LB_INVALID_ARGUMENT, "%s: rotated dims must be even, 2 to head_dim", what);
  if (r.pairs > LB_PAIRS_NEIGHBOURS) return fail(LB_INVALID_ARGUMENT, "%s: unknown pairs %u", what, r.pairs);
  return std::isfinite(r.scale) ? LB_OK : fail(LB_INVALID_ARGUMENT, "%s: the rotation's scale must be finite", what);
}

inline Turn turn_params(const lb_rotation &r) { return {r.frequencies, (int)r.dims, r.pairs == LB_PAIRS_NEIGHBOURS, r.scale}; }

template <class T>
Rows<T> strided(const lb_rows &r) {
  return {static_cast<T *>(r.data), (long long)r.batch_stride, (long long)r.row_stride, (long long)r.head_stride};
}

inline bool same_rows(const lb_rows &a, const lb_rows &b, int64_t batch, int64_t seq, int64_t heads) {
  return a.data == b.data && (batch == 1 || a.batch_stride == b.batch_stride) && (seq == 1 || a.row_stride == b.row_stride) &&
         (heads == 1 || a.head_stride == b.head_stride);
}

}  // namespace abi
}  // namespace lb
