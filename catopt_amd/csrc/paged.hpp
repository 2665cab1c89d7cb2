// What the kernels of the paged cache share: the page arithmetic.
#pragma once
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

inline bool strides_fit(const int64_t* s, int n, int64_t step) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % step) return false;
  return true;
}

}  // namespace catopt
