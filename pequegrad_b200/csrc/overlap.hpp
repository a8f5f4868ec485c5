// Do strided views share bytes? Asked on the host of the tensors that a call writes: threads that write one byte race.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace pgb {

// A run of `len` bytes at `base`, repeated over up to four dims (strides in bytes, not negative).
struct ByteView {
  uintptr_t base;
  int64_t len;
  __int128 end;  // behind the last byte
  int dims = 0;
  int64_t n[4], stride[4];

  ByteView(uintptr_t at = 0, int64_t bytes = 0) : base(at), len(bytes), end((__int128)at + bytes) {}
  void add(int64_t extent, int64_t step) {
    if (extent <= 0) len = 0;
    if (extent > 1) {
      end += (__int128)(extent - 1) * step;
      n[dims] = extent;
      stride[dims++] = step;
    }
  }
  bool operator==(const ByteView &o) const {
    if (base != o.base || len != o.len || dims != o.dims) return false;
    for (int i = 0; i < dims; ++i)
      if (n[i] != o.n[i] || stride[i] != o.stride[i]) return false;
    return true;
  }
};

// Is there a sum at + c_0 s_0 + c_1 s_1 + .. between `low` and `high` (both excluded), lo_i <= c_i <= hi_i? Strides in descending
// order. At each dim only those c are tried from which the rest can still reach; in views whose dims nest that is one or two. A
// search that does not end in a few thousand steps counts as yes.
struct StrideSums {
  int dims = 0;
  int64_t s[8], lo[8], hi[8];
  __int128 low, high;
  int budget = 4096;

  void add(int64_t stride, int64_t from, int64_t to) {
    int i = 0;
    while (i < dims && s[i] > stride) ++i;
    if (i < dims && s[i] == stride) {
      lo[i] += from;
      hi[i] += to;
      return;
    }
    for (int k = dims++; k > i; --k) { s[k] = s[k - 1]; lo[k] = lo[k - 1]; hi[k] = hi[k - 1]; }
    s[i] = stride;
    lo[i] = from;
    hi[i] = to;
  }
  static __int128 div_down(__int128 a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
  bool any(__int128 at, int dim = 0) {
    if (--budget < 0) return true;
    if (dim == dims) return low < at && at < high;
    if (s[dim] == 0) return any(at, dim + 1);
    __int128 least = 0, most = 0;  // of the dims behind this one
    for (int i = dim + 1; i < dims; ++i) { least += (__int128)lo[i] * s[i]; most += (__int128)hi[i] * s[i]; }
    const __int128 from = std::max<__int128>(lo[dim], div_down(low - at - most, s[dim]) + 1);
    const __int128 to = std::min<__int128>(hi[dim], div_down(high - 1 - at - least, s[dim]));
    for (__int128 c = from; c <= to; ++c)
      if (any(at + c * s[dim], dim + 1)) return true;
    return false;
  }
};

// Of a tensor descriptor whose last dim is contiguous, `es` bytes an element, up to five dims.
template <typename Tensor>
inline ByteView view_of(const Tensor &t, int es) {
  ByteView v(reinterpret_cast<uintptr_t>(t.data), es * t.shape[t.ndim - 1]);
  for (int i = 0; i + 1 < t.ndim; ++i) v.add(t.shape[i], t.stride_bytes[i]);
  return v;
}

inline bool views_share(const ByteView &a, const ByteView &b) {
  if (a.end <= (__int128)b.base || b.end <= (__int128)a.base || a.len <= 0 || b.len <= 0) return false;  // the usual case
  StrideSums d;
  for (int i = 0; i < a.dims; ++i) d.add(a.stride[i], 0, a.n[i] - 1);
  for (int i = 0; i < b.dims; ++i) d.add(b.stride[i], 1 - b.n[i], 0);
  d.low = -(__int128)a.len;
  d.high = b.len;
  return d.any((__int128)a.base - (__int128)b.base);
}

inline bool view_overlaps_itself(const ByteView &a) {
  if (a.len <= 0) return false;
  for (int k = 0; k < a.dims; ++k) {  // two places that differ in dim k, and in the later dims as they like
    StrideSums d;
    d.low = -(__int128)a.len;
    d.high = a.len;
    for (int i = k + 1; i < a.dims; ++i) d.add(a.stride[i], 1 - a.n[i], a.n[i] - 1);
    d.add(a.stride[k], 1, a.n[k] - 1);
    // merged with a dim of the same stride, c_k = 1 and c_i = -1 cancel: that is an overlap, and the sum finds it
    if (d.any(0)) return true;
  }
  return false;
}

}  // namespace pgb
