// What the kernels of the paged cache share: the page arithmetic.
#pragma once
#include <initializer_list>

#include "common.hpp"

namespace catopt {

// Division of 0 <= n < 2^31 by a positive divisor below 2^31 as a multiply and
// a shift: with L = ceil(log2 d), m = ceil(2^(31 + L) / d) < 2^32 exceeds the
// quotient's slope by e / 2^(31 + L), e < 2^L, so n e < 2^(31 + L) and the
// floor is exact.
struct FastDiv {
  uint32_t d, m, shift;
  static FastDiv of(int64_t d) {
    FastDiv f;
    f.d = (uint32_t)d;
    uint32_t l = 0;
    while ((1ull << l) < (uint64_t)d) ++l;
    f.shift = 31 + l;
    f.m = (uint32_t)(((1ull << f.shift) + (uint64_t)d - 1) / (uint64_t)d);
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> shift); }
};

// One tensor of pages: [page][head][slot][d], strides in elements.
struct Pages {
  const void* p;
  int64_t s_page, s_head, s_slot;
};

// The rows [row0, row0 + nq) of sequence b among N: whatever starts holds, they
// lie inside the operands.
__device__ __forceinline__ void seq_rows(const int32_t* starts, int b, int64_t N, int& row0, int& nq) {
  const int n = (int)N;  // N <= 2^30
  row0 = min(max(starts[b], 0), n);
  nq = max(min(max(starts[b + 1], 0), n) - row0, 0);
}

// Strides as the kernels take them: none negative, multiples of `step`; that of
// an axis of one entry, which may be anything, as 0.
struct Strides {
  int64_t s[16];
  bool fit = true;
  Strides(const int64_t* in, std::initializer_list<int64_t> extents, int64_t step) {
    int i = 0;
    for (const int64_t n : extents) {
      s[i] = n > 1 ? in[i] : 0;
      if (s[i] < 0 || s[i] % step) fit = false;
      ++i;
    }
  }
};

// A tensor's layout for the checks of what may overlap what: up to four axes,
// extents and strides in elements, and the size of one.
struct Layout {
  const void* p;
  int n;
  int64_t extent[4], stride[4], size;

  bool empty() const {
    for (int i = 0; i < n; ++i)
      if (extent[i] < 1) return true;
    return !p;
  }
  uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
  // One byte behind the last element.
  uintptr_t end() const {
    int64_t last = 0;
    for (int i = 0; i < n; ++i) last += (extent[i] - 1) * stride[i];
    return begin() + (uintptr_t)((last + 1) * size);
  }
  // Whether two elements share memory (an expanded tensor).
  bool folded() const {
    if (empty()) return false;
    int64_t s[4], e[4];
    int m = 0;
    for (int i = 0; i < n; ++i) {
      if (extent[i] < 2) continue;
      int at = m++;
      for (; at > 0 && s[at - 1] > stride[i]; --at) s[at] = s[at - 1], e[at] = e[at - 1];
      s[at] = stride[i], e[at] = extent[i];
    }
    int64_t need = 1;
    for (int i = 0; i < m; ++i) {
      if (s[i] < need) return true;
      need = s[i] * e[i];
    }
    return false;
  }
  bool overlaps(const Layout& o) const { return !empty() && !o.empty() && begin() < o.end() && o.begin() < end(); }
  bool same(const Layout& o) const {
    if (p != o.p) return false;
    for (int i = 0; i < n; ++i)
      if (extent[i] > 1 && stride[i] != o.stride[i]) return false;
    return true;
  }
};

inline Layout layout3(const void* p, int64_t size, int64_t a, int64_t sa, int64_t b, int64_t sb, int64_t c) {
  return Layout{p, 3, {a, b, c, 1}, {sa, sb, 1, 1}, size};
}
inline Layout layout_pages(const void* p, int64_t size, int64_t n_pages, int64_t H, int64_t page, int64_t d,
                           const int64_t* s) {
  return Layout{p, 4, {n_pages, H, page, d}, {s[0], s[1], s[2], 1}, size};
}

}  // namespace catopt
