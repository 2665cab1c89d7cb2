// What the kernels of token sampling share: a call's arguments, a row's settings
// and the fixed-point weights.
#pragma once
#include "common.hpp"

namespace catopt {

// Weights exp((x - max) / T) lie on a grid of 16 steps to a factor of 2: with y =
// x 16 log2(e) / T and n its whole part, a logit belongs to the bin n and weighs
// 2^(n / 16) 2^((y - n) / 16).  The second factor, from 1 to 1.045, is rounded to 34
// bits behind the point: a bin's weight is then a sum of integers, the same in
// every order, whichever chunk of the row a logit lies in.  What a choice can be off
// by is what such sums are off by, 2^-35 of a weight at random and 2^-38 with one
// sign: a step of u is 2^-24.  A bin 768 steps below the largest logit's weighs
// 2^-48 of it or less and counts as nothing.
//
// A chunk's bin holds the sum below bit 49 and the number of logits above.
constexpr int kBins = 768;
constexpr int kPoint = 34, kCount = 49;
constexpr int kMaxChunk = 1 << 14;        // its sum stays below 2^(14 + 34.07), its number fits 15 bits
constexpr int64_t kMaxVocab = 1LL << 21;
// Sums over bins are in units of 2^-42 of bin 0's weight: below 2^(21 + 42.07).
constexpr int kUnits = 42;

struct SampleArgs {
  const void* x;
  int64_t ld, ld_probs;
  int V, B, chunks;
  // a row's own setting, else the call's
  const float *t_row, *p_row, *low_row;
  const int32_t* k_row;
  double t, p, low;
  int64_t k;
  const float* u;
  int64_t* tokens;
  float *logprobs, *probs;
  struct ChunkHead* heads;  // [B][chunks]
  uint64_t* bins;           // [B][chunks][kBins]
  struct RowState* rows;    // [B], for the probabilities
};

struct ChunkHead {
  float max;
  int32_t first;  // greedy rows: where the largest logit is first
  int32_t nan, pad;
};

// What the probabilities of a row are worked out from.
struct RowState {
  double c, low, log2_total;  // y = c x; the least y; log2 of the kept weights
  uint64_t cut_at;            // in the cut's bin the last place that is kept
  int32_t cut, token;         // the last bin that is kept (some of it); kOneHot, kNone: the token alone, NaN
  float max, floor;           // the largest logit; nothing below the floor is kept
};
constexpr int kOneHot = -1, kNone = -2;

struct Settings {
  double t, p, low;
  int64_t k;
  bool greedy, valid;
};

__device__ __forceinline__ Settings settings(const SampleArgs& a, int row) {
  Settings s;
  s.t = a.t_row ? (double)a.t_row[row] : a.t;
  s.p = a.p_row ? (double)a.p_row[row] : a.p;
  s.low = a.low_row ? (double)a.low_row[row] : a.low;
  s.k = a.k_row ? (int64_t)a.k_row[row] : a.k;
  s.valid = s.t >= 0;
  s.greedy = s.t == 0 || s.k == 1;
  if (s.k <= 0 || s.k >= a.V) s.k = 0;  // all
  return s;
}

// y's factor: at most 2^40 for the largest logit, where all that is not equal to it
// lies far behind the last bin, so that n is exact; above 0 for -inf to stay -inf.
__device__ __forceinline__ double factor(double t, float max) {
  return fmax(fmin(16 * 1.4426950408889634 / t, 0x1p40 / fmax(fabs((double)max), 0x1p-120)), 0x1p-160);
}

__device__ __forceinline__ uint64_t bits_of(double v) { return __builtin_bit_cast(uint64_t, v); }

// A row's grid: y, less a whole number near the largest logit's, on top of 1.5 2^20.
// That sum's upper word then has y's whole part and its lower word the 32 bits behind
// the point: a bin and a logit's part of it cost one fused multiply-add and one
// subtraction.  The constants of a weight stay in registers: left to itself the
// compiler sets them anew for every logit of an unrolled loop, a third of its
// instructions.
struct Grid {
  double c, shift, top;  // y's factor; what is added; the largest logit's whole part
  uint32_t ref;          // and its upper word
  double s4, s3, s2, s1, s0;

  __device__ __forceinline__ Grid(double c_, float max) : c(c_) {
    const double n = __builtin_fma((double)max, c, 0x1.8p52) - 0x1.8p52;
    shift = 0x1.8p20 - n;
    ref = (uint32_t)(bits_of(on(max)) >> 32);
    top = n + (double)(int)(ref - 0x41380000u);
    // Of 2^(part / 16), part from 0 to 1 in steps of 2^-32: the polynomial of the
    // fourth power that Chebyshev's expansion gives, off by 2^-38.5 of it at most (one
    // of the third by 2^-29.7), with 2^52 to make the sum's mantissa an integer.
    constexpr double one = 1LL << kPoint, p = 0x1p-32;
    s4 = one * p * p * p * p * 1.499781553911453e-07, s3 = one * p * p * p * 1.3547981600582377e-05;
    s2 = one * p * p * 0.0009383858041510473, s1 = one * p * 0.04332169865843112, s0 = one * 1.000000000002533 + 0x1p52;
    asm("" : "+s"(s4), "+v"(s3), "+s"(s2), "+s"(s1), "+s"(s0));
  }
  __device__ __forceinline__ double on(float x) const { return __builtin_fma((double)x, c, shift); }
  // Bins from the largest logit's down to this one's; a large number for one far below, -inf or a NaN.
  __device__ __forceinline__ uint32_t bin(double on) const { return ref - (uint32_t)(bits_of(on) >> 32); }
  static __device__ __forceinline__ uint32_t part(double on) { return (uint32_t)bits_of(on); }
  // 2^(part / 16) in fixed point.
  __device__ __forceinline__ uint64_t weight(uint32_t part) const {
    const double u = (double)part;
    double s = __builtin_fma(s4, u, s3);
    s = __builtin_fma(s, u, s2);
    s = __builtin_fma(s, u, s1);
    s = __builtin_fma(s, u, s0);
    return bits_of(s) & 0xfffffffffffffull;  // below 2^35
  }
  // log2 of a weight to the largest logit's bin's, times 16.
  static __device__ __forceinline__ double log_weight(int bin, uint32_t part) { return (double)part * 0x1p-32 - bin; }
};

// The order of a row, as ascending numbers: the largest logit first, the lowest
// index first among equals (-0 as 0).
__device__ __forceinline__ uint64_t place(float x, int i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  const uint32_t key = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return (uint64_t)~key << 32 | (uint32_t)i;
}
__device__ __forceinline__ float logit_of(uint64_t place) {
  const uint32_t key = ~(uint32_t)(place >> 32);
  return __builtin_bit_cast(float, key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// A row in aligned pieces of 16 bytes, W logits each, and the few logits before the
// first and behind the last of them.
template <typename T>
struct RowReader {
  static constexpr int W = 16 / sizeof(T);
  const T* row;
  int V, head, pieces;

  __device__ __forceinline__ RowReader(const SampleArgs& a, int r)
      : row(static_cast<const T*>(a.x) + (int64_t)r * a.ld), V(a.V) {
    const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min(shift ? W - shift : 0, V);
    pieces = (V - head) / W;
  }
  __device__ __forceinline__ int first(int piece) const { return head + piece * W; }
  // -inf behind the last piece.
  __device__ __forceinline__ u32x4 load(int piece) const {
    const uint32_t none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    u32x4 w = {none, none, none, none};
    if (piece < pieces) w = *reinterpret_cast<const u32x4*>(row + first(piece));
    return w;
  }
  // Logit e of a piece.
  static __device__ __forceinline__ float at(const u32x4& w, int e) {
    const uint32_t word = sizeof(T) == 4 ? w[e] : w[e / 2];
    return __builtin_bit_cast(float, sizeof(T) == 4 ? word : e & 1 ? word & 0xffff0000u : word << 16);
  }
  // Those outside the pieces, less than 2 W.
  __device__ __forceinline__ int edges() const { return V - pieces * W; }
  __device__ __forceinline__ int edge(int i) const { return i < head ? i : pieces * W + i; }
  __device__ __forceinline__ float value(int i) const { return load_f32(row, i); }
};

// +inf as the largest finite number (one instruction: fminf makes NaNs quiet first).
__device__ __forceinline__ float finite_top(float x) {
  float y;
  asm("v_min_f32 %0, %1, %2" : "=v"(y) : "s"(0x1.fffffep127f), "v"(x));
  return y;
}

}  // namespace catopt
