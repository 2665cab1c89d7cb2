// The next token of each row of logits: temperature, top-k, top-p, min-p and one
// random number.
//
// In the order of a row (the largest logit first) what is kept is a prefix, and the
// token is the first kept one whose running sum of weights passes u times the kept
// weights.  So nothing is sorted: a chunk's workgroup adds its logits' weights up in
// bins (one read of the row), and a row's workgroup finds the bins in which the
// borders and the token lie, reads the row again for the logits of those alone, and
// narrows them down to at most 64, which one wave ranks.
#include "sampling.hpp"

namespace catopt {
namespace {

// ---------------------------------------------------------------- chunks

constexpr int CT = 512;

template <typename T, int EPT>
__global__ __launch_bounds__(CT) void sample_chunks(SampleArgs a) {
  constexpr int W = RowReader<T>::W, P = EPT / W;
  __shared__ uint64_t weights[kBins];
  __shared__ uint32_t counts[kBins];
  __shared__ float maxima[CT / 64];
  __shared__ int firsts[CT / 64], nans[CT / 64];
  const int row = (int)(blockIdx.x / (uint32_t)a.chunks), chunk = (int)(blockIdx.x - (uint32_t)row * a.chunks);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const RowReader<T> r(a, row);
  const int piece0 = chunk * (CT * P) + tid;
  u32x4 w[P];
#pragma unroll
  for (int j = 0; j < P; ++j) w[j] = r.load(piece0 + j * CT);
  const Settings s = settings(a, row);
  const bool binned = s.valid && !s.greedy, counted = binned && s.k;
  if (binned)
    for (int i = tid; i < kBins; i += CT) weights[i] = 0, counts[i] = 0;
  float m = -__builtin_inff();
  bool nan = false;
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float x = r.at(w[j], e);
      nan |= x != x;
      m = fmaxf(m, x);
    }
  m = finite_top(m);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const bool any_nan = __ballot(nan) != 0;
  if (lane == 0) maxima[wave] = m, nans[wave] = any_nan;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < CT / 64; ++i) m = fmaxf(m, maxima[i]);
  ChunkHead* head = a.heads + (int64_t)row * a.chunks + chunk;
  if (s.greedy) {
    int first = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int e = W - 1; e >= 0; --e)
        if (finite_top(r.at(w[j], e)) == m) first = min(first, r.first(piece0 + j * CT) + e);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
    if (lane == 0) firsts[wave] = first;
    __syncthreads();
  }
  if (tid == 0) {
    ChunkHead h{m, 0x7fffffff, 0, 0};
    for (int i = 0; i < CT / 64; ++i) {
      h.nan |= nans[i];
      if (s.greedy) h.first = min(h.first, firsts[i]);
    }
    *head = h;
  }
  if (!binned || m == -__builtin_inff()) return;
  const double c = factor(s.t, m);
  double rest;
  const double ref = grid(m, c, rest);
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const double d = ref - grid(finite_top(r.at(w[j], e)), c, rest);
      if (d < kBins) {  // not so for -inf, nor where T is infinite and that a NaN
        const int bin = (int)d;
        atomicAdd(reinterpret_cast<unsigned long long*>(weights + bin), (unsigned long long)fixed(rest));
        if (counted) atomicAdd(counts + bin, 1u);
      }
    }
  __syncthreads();
  const int64_t at = ((int64_t)row * a.chunks + chunk) * kBins;
  for (int i = tid; i < kBins; i += CT) {
    a.weights[at + i] = weights[i];
    if (counted) a.counts[at + i] = counts[i];
  }
}

// ------------------------------------------------------------------ rows

constexpr int RT = 1024, WAVES = RT / 64;
constexpr int kList = 8192;   // logits of a row that are kept in LDS
constexpr int kParts = 256;   // of a range
constexpr int kMaxChunks = 520;

// What one step of a search adds up.  Three of them take turns: a step clears the
// next one's, which was last read before the barrier that ended the step before,
// so that a step is one barrier.
struct Step {
  uint64_t weight[kParts];
  uint64_t last[64];
  uint32_t n[kParts];
  uint32_t count;
};

struct RowLds {
  uint64_t cum[kBins];  // weights up to a bin's end, in units of 2^-42 of bin 0's
  uint64_t list[kList];
  Step steps[3];
  uint64_t wave_sums[WAVES];
  uint32_t cum_n[kBins];  // logits up to it: exactly with a top-k, else at most
  uint32_t wave_counts[WAVES];
  int off[kMaxChunks];  // a chunk's first bin among the row's
};

// (min and max of the headers take 64-bit integers as doubles.)
__device__ __forceinline__ uint64_t least_of(uint64_t a, uint64_t b) { return a < b ? a : b; }

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32 | (uint32_t)__shfl((int)(uint32_t)v, lane, 64);
}
// Inclusive sums over the wave.
__device__ __forceinline__ uint64_t scan_u64(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = shfl_u64(v, max(lane - o, 0));
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ uint32_t scan_u32(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ double scan_f64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// The wave's places (~0 behind the last) in ascending order, lane by lane.
__device__ __forceinline__ uint64_t sorted(uint64_t mine, int n) {
  int rank = 0;
  for (int j = 0; j < n; ++j) rank += shfl_u64(mine, j) < mine;
  if ((int)(threadIdx.x & 63) >= n) rank = threadIdx.x & 63;
  const uint32_t hi = __builtin_amdgcn_ds_permute(4 * rank, (int)(mine >> 32));
  const uint32_t lo = __builtin_amdgcn_ds_permute(4 * rank, (int)(uint32_t)mine);
  return (uint64_t)hi << 32 | lo;
}

// What a border or the token is looked for by: the logit at a rank, or the first
// whose running sum of weights reaches or passes a number.
enum Find { kRank, kReaches, kPasses };
__device__ __forceinline__ bool meets(Find f, double target, uint64_t sum, uint32_t n) {
  return f == kRank ? (double)n > target : f == kReaches ? (double)sum >= target : (double)sum > target;
}

// Bin b's weight to bin 0's.
__device__ __forceinline__ double scale_of(int b) { return exp2(-(double)b / 16); }

struct Bins {
  int first, last;
  __device__ __forceinline__ bool has(int b) const { return b >= first && b <= last; }
};
constexpr Bins kNoBins{1, 0};

// A row's search.  Every wave comes to the same decisions, from what is in LDS.
template <typename T>
struct Search {
  RowLds& s;
  const RowReader<T> r;
  double c, ref;
  int step = 0;
  uint32_t n_list = 0;
  Bins listed = kNoBins, listed2 = kNoBins;  // the list holds all their logits

  __device__ __forceinline__ int bin_of(float x, double& rest) const {
    const double d = ref - grid(x, c, rest);
    return d < kBins ? (int)d : kBins;
  }

  // Numbers that no logit of bins up to b is below, or from b on above.
  __device__ __forceinline__ float floor_of(int b) const {
    const float f = (float)((ref - b - 0.5) / c);
    return f - fabsf(f) * 0x1p-22f - 0x1p-140f;
  }
  __device__ __forceinline__ float top_of(int b) const {
    const float f = (float)((ref - b + 0.5) / c);
    return f + fabsf(f) * 0x1p-22f + 0x1p-140f;
  }

  __device__ __forceinline__ Step& begin() {
    Step& next = s.steps[(step + 1) % 3];
    if (threadIdx.x < kParts) next.weight[threadIdx.x] = 0, next.n[threadIdx.x] = 0;
    if (threadIdx.x == 0) next.count = 0;
    return s.steps[step++ % 3];
  }

  // f(place, rest) for the row's logits in either of the bins.
  template <typename F>
  __device__ __forceinline__ void scan_row(Bins a, Bins b, F f) const {
    constexpr int U = 4;
    // most logits fall out by two comparisons; the others' bins are worked out
    const float lo = floor_of(a.last), hi = top_of(a.first), lo2 = floor_of(b.last), hi2 = top_of(b.first);
    const bool two = b.first <= b.last;
    const int n = r.pieces();
#pragma unroll 1
    for (int p0 = threadIdx.x; p0 < n; p0 += U * RT) {
      u32x4 w[U];
#pragma unroll
      for (int j = 0; j < U; ++j) w[j] = r.load(p0 + j * RT);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < RowReader<T>::W; ++e) {
          const float x = r.at(w[j], e);
          some |= ((x >= lo && x <= hi) || (two && x >= lo2 && x <= hi2)) ? 1u << e : 0u;
        }
        while (some) {
          const int e = __builtin_ctz(some);
          some &= some - 1;
          float x = r.at(w[j], 0);
#pragma unroll
          for (int i = 1; i < RowReader<T>::W; ++i) x = i == e ? r.at(w[j], i) : x;
          x = finite_top(x);
          double rest;
          const int bin = bin_of(x, rest);
          if (a.has(bin) || b.has(bin)) f(place(x, r.first(p0 + j * RT) + e), rest);
        }
      }
    }
  }

  // The logits of a range of places of those bins into the list, as far as it
  // holds them; their number.
  __device__ __forceinline__ uint32_t gather(Bins a, Bins b, uint64_t lo, uint64_t hi) {
    Step& t = begin();
    scan_row(a, b, [&](uint64_t at, double) {
      if (at < lo || at > hi) return;
      const uint32_t i = atomicAdd(&t.count, 1u);
      if (i < kList) s.list[i] = at;
    });
    __syncthreads();
    return t.count;
  }

  // The same to be searched in afterwards, if it holds them.
  __device__ __forceinline__ void list_bins(Bins a, Bins b) {
    n_list = gather(a, b, 0, ~0ull);
    const bool all = n_list <= kList;
    listed = all ? a : kNoBins, listed2 = all ? b : kNoBins;
  }

  // The first bin whose running sum (or count) meets the target, kBins - 1 where none does.
  __device__ __forceinline__ int find_bin(Find find, double target) const {
    const int lane = threadIdx.x & 63, group = 64 * min(lane, kBins / 64 - 1);
    const uint64_t ends = __ballot(lane < kBins / 64 && meets(find, target, s.cum[group + 63], s.cum_n[group + 63]));
    if (!ends) return kBins - 1;
    const int first = 64 * __builtin_ctzll(ends);
    return first + __builtin_ctzll(__ballot(meets(find, target, s.cum[first + lane], s.cum_n[first + lane])));
  }

  // Of bin b, the logit that `find` names by `target` (a rank or a sum within the
  // bin): its place and the sum up to it; the last one where none does.
  __device__ __forceinline__ uint64_t resolve(int b, Find find, double target, uint64_t& sum) {
    const int lane = threadIdx.x & 63;
    const Bins one{b, b};
    uint64_t lo = place(top_of(b), 0), hi = place(floor_of(b), -1), before = 0;
    uint32_t n_before = 0, n = s.cum_n[b] - (b ? s.cum_n[b - 1] : 0);
    bool list = listed.has(b) || listed2.has(b), own = false;  // own: the list is this call's, and holds the range alone
    for (;;) {
      if (!list && n <= kList) {
        listed = listed2 = kNoBins;
        n = n_list = gather(one, kNoBins, lo, hi);
        list = own = true;
      }
      // one key alone: its indexes end with the row
      if (lo >> 32 == hi >> 32) hi = least_of(hi, (hi & ~0xffffffffull) | (uint32_t)(r.V - 1));
      const bool few = n <= 64;
      const int bits = 64 - __builtin_clzll((hi - lo) | 1), shift = max(bits - 8, 0);
      Step& t = begin();
      auto take = [&](uint64_t at, double rest) {
        if (at < lo || at > hi) return;
        if (few) {
          t.last[atomicAdd(&t.count, 1u) & 63] = at;
        } else {
          const int i = (int)((at - lo) >> shift);
          atomicAdd(reinterpret_cast<unsigned long long*>(t.weight + i), (unsigned long long)fixed(rest));
          atomicAdd(t.n + i, 1u);
        }
      };
      if (list) {
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n_list; i += RT) {
          const uint64_t at = s.list[i];
          double rest;
          if (bin_of(logit_of(at), rest) == b) take(at, rest);
        }
      } else {
        scan_row(one, kNoBins, take);
      }
      __syncthreads();
      if (few) {  // a wave puts them in order
        const int m = min((int)t.count, 64);
        const uint64_t at = sorted(lane < m ? t.last[lane] : ~0ull, m);
        double rest;
        bin_of(logit_of(at), rest);
        const uint64_t upto = scan_u64(lane < m ? fixed(rest) : 0) + before;
        const uint64_t some = __ballot(lane < m && meets(find, target, upto, n_before + lane + 1));
        const int from = some ? __builtin_ctzll(some) : max(m - 1, 0);
        sum = shfl_u64(upto, from);
        if (own) listed = listed2 = kNoBins;
        return shfl_u64(at, from);
      }
      // four parts a lane: the part that the logit is in, the last that holds one where none meets the target
      uint64_t w[4], all = 0;
      uint32_t k[4], all_n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = t.weight[4 * lane + i], k[i] = t.n[4 * lane + i];
        all += w[i], all_n += k[i];
      }
      uint64_t upto = scan_u64(all) - all + before, at_sum = 0;
      uint32_t upto_n = scan_u32(all_n) - all_n + n_before, at_n = 0, here = 0;
      int at = -1;
      bool met = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k[i] && !met) {
          at = 4 * lane + i, at_sum = upto, at_n = upto_n, here = k[i];
          met = meets(find, target, upto + w[i], upto_n + k[i]);
        }
        upto += w[i], upto_n += k[i];
      }
      const uint64_t some = __ballot(met), held = __ballot(at >= 0);
      const int from = some ? __builtin_ctzll(some) : 63 - __builtin_clzll(held | 1);
      const int part = max(__shfl(at, from, 64), 0);
      lo += (uint64_t)part << shift;
      hi = least_of(hi, lo + ((1ull << shift) - 1));
      before = shfl_u64(at_sum, from), n_before = __shfl(at_n, from, 64), n = __shfl(here, from, 64);
    }
  }
};

template <typename T>
__global__ __launch_bounds__(RT) void sample_rows(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  RowLds& s = *reinterpret_cast<RowLds*>(lds);
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Settings set = settings(a, row);
  const ChunkHead* heads = a.heads + (int64_t)row * a.chunks;
  float m = -__builtin_inff();
  int nan = 0;
  for (int i = lane; i < a.chunks; i += 64) {
    const ChunkHead h = heads[i];
    m = fmaxf(m, h.max);
    nan |= h.nan;
  }
  const float u_row = a.u[row];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const bool valid = set.valid && __ballot(nan != 0) == 0 && m != -__builtin_inff();
  if (!valid || set.greedy) {
    int first = 0x7fffffff;
    if (valid)
      for (int i = lane; i < a.chunks; i += 64) first = heads[i].max == m ? min(first, heads[i].first) : first;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
    if (tid == 0) {
      a.tokens[row] = valid ? first : -1;
      a.logprobs[row] = valid ? 0.f : __builtin_nanf("");
      if (a.rows) a.rows[row] = RowState{0, 0, 0, 0, 0, valid ? kOneHot : kNone, first};
    }
    return;
  }
  const double c = factor(set.t, m);
  double rest;
  const double ref = grid(m, c, rest);
  Search<T> find{s, RowReader<T>(a, row), c, ref};
  // ---- the row's bins from the chunks'
  for (int i = tid; i < a.chunks; i += RT) {
    const float cm = heads[i].max;
    // by the row's factor: it is the chunk's too wherever the chunk has a bin of the row's
    const double d = cm == -__builtin_inff() ? kBins : ref - grid(cm, c, rest);
    s.off[i] = d < kBins ? max((int)d, 0) : kBins;
  }
  if (tid < kParts) s.steps[0].weight[tid] = 0, s.steps[0].n[tid] = 0;
  if (tid == 0) s.steps[0].count = 0;
  __syncthreads();
  const bool counted = set.k != 0;
  uint64_t w = 0;
  uint32_t n = 0;
  if (tid < kBins) {
    const uint64_t* ws = a.weights + (int64_t)row * a.chunks * kBins + tid;
    const uint32_t* ns = a.counts + (int64_t)row * a.chunks * kBins + tid;
#pragma unroll 4
    for (int i = 0; i < a.chunks; ++i) {
      const int o = s.off[i];
      const bool in = tid >= o;
      w += in ? ws[(int64_t)i * kBins - o] : 0;
      if (counted) n += in ? ns[(int64_t)i * kBins - o] : 0;
    }
    // a logit weighs at least 0.978 in its bin
    if (!counted) n = (uint32_t)((double)w * (1.0 / (0.978 * (1LL << kPoint)))) + (w != 0);
    w = (uint64_t)rint((double)w * scale_of(tid));
  }
  {
    const uint64_t sw = scan_u64(w);
    const uint32_t sn = scan_u32(n);
    if (lane == 63) s.wave_sums[wave] = sw, s.wave_counts[wave] = sn;
    __syncthreads();
    uint64_t bw = 0;
    uint32_t bn = 0;
    for (int i = 0; i < wave; ++i) bw += s.wave_sums[i], bn += s.wave_counts[i];
    if (tid < kBins) s.cum[tid] = bw + sw, s.cum_n[tid] = bn + sn;
  }
  __syncthreads();
  // ---- the kept prefix: up to `cut_at` in bin `cut`, `total` in all
  // below 1 by half a step of fp32 at least, so that the product stays below the total; a NaN counts as 0
  const double u = fmin(fmax((double)u_row, 0.0), 1 - 0x1p-25);
  int cut = kBins - 1;
  uint64_t cut_at = ~0ull, total = s.cum[kBins - 1];
  bool by_rank = counted && s.cum_n[kBins - 1] > set.k, by_sum = set.p < 1, by_low = set.low > 0;
  const double low = by_low ? (double)m * c + 16 * log2(fmin(set.low, 1.0)) : -__builtin_inf();
  const double low_bin = by_low ? ref - rint(low) : kBins;
  auto before = [&](int b) { return b > 0 ? s.cum[b - 1] : 0ull; };
  auto before_n = [&](int b) { return b > 0 ? s.cum_n[b - 1] : 0u; };
  auto within = [&](int b, uint64_t sum) { return before(b) + (uint64_t)rint((double)sum * scale_of(b)); };
  if (by_rank || by_sum || by_low) {
    if (by_rank) cut = find.find_bin(kRank, (double)(set.k - 1));
    int end = by_rank || !by_sum ? cut : find.find_bin(kReaches, set.p * (double)total);
    // a border behind min-p's does nothing, but for a rank's that says what top-p is a share of
    by_low = low_bin <= end;
    if (low_bin < end && !(by_rank && by_sum)) by_rank = by_sum = false, end = (int)low_bin;
    if (s.cum_n[end] <= kList) {
      find.list_bins({0, end}, kNoBins);
      if (find.n_list <= 64) {
        // all that may be kept is in one wave: the definition, lane by lane
        const int n_all = (int)find.n_list;
        const uint64_t at = sorted(lane < n_all ? s.list[lane] : ~0ull, n_all);
        const int bin = find.bin_of(logit_of(at), rest);
        const double sums = scan_f64(lane < n_all ? (double)fixed(rest) * scale_of(bin) : 0);
        const double whole = by_rank ? __shfl(sums, (int)set.k - 1, 64) : (double)total;
        bool kept = lane < (by_rank ? (int)set.k : n_all);
        if (by_sum) {
          const uint64_t reach = __ballot(kept && sums >= set.p * whole);
          if (reach) kept = lane <= __builtin_ctzll(reach);
        }
        if (by_low) kept = kept && (double)logit_of(at) * c >= low;
        const int last = 63 - __builtin_clzll(__ballot(kept) | 1);
        const double kept_sum = __shfl(sums, last, 64);
        const uint64_t pass = __ballot(lane <= last && sums > u * kept_sum);
        const int from = pass ? __builtin_ctzll(pass) : last;
        const double log2_total = log2(kept_sum) - kPoint;
        if (wave == 0 && lane == from) {
          a.tokens[row] = (int64_t)(uint32_t)at;
          a.logprobs[row] = (float)(((rest - bin) / 16 - log2_total) * 0.6931471805599453);
        }
        if (wave == 0 && lane == last && a.rows) a.rows[row] = RowState{c, ref, low, log2_total, at, bin, 0};
        return;
      }
    } else if (!by_rank) {
      // the border lies in bin `end`, the token where u says for a whole between the sums before and behind it: both
      // are read at once if they fit
      const Bins pick{find.find_bin(kPasses, u * (double)before(end)), min(find.find_bin(kPasses, u * (double)s.cum[end]), end - 1)};
      const uint32_t here = s.cum_n[end] - before_n(end);
      const uint32_t there = pick.first <= pick.last ? s.cum_n[pick.last] - before_n(pick.first) : 0;
      if (here + there <= kList) find.list_bins({end, end}, pick);
    }
    uint64_t sum;
    if (by_rank) {
      if (s.cum_n[cut] == set.k) {
        total = s.cum[cut];
      } else {
        cut_at = find.resolve(cut, kRank, (double)(set.k - 1 - before_n(cut)), sum);
        total = within(cut, sum);
      }
    }
    if (by_sum) {
      const double target = set.p * (double)total;
      const int b = min(find.find_bin(kReaches, target), cut);
      const uint64_t at = find.resolve(b, kReaches, (target - (double)before(b)) / scale_of(b), sum);
      if (b < cut || at < cut_at) cut = b, cut_at = at, total = within(b, sum);
    }
    if (by_low && low_bin <= cut) {
      // of the border's bin those whose y is not below it
      const int b = (int)low_bin;
      if (!find.listed.has(b)) find.list_bins({b, b}, kNoBins);
      Step& t = find.begin();
      uint64_t mine = 0;
      auto take = [&](float x, uint64_t at, double rs) {
        if ((double)x * c >= low && (b < cut || at <= cut_at)) mine += fixed(rs);
      };
      if (find.listed.has(b)) {
        for (uint32_t i = tid; i < find.n_list; i += RT) {
          const float x = logit_of(s.list[i]);
          if (find.bin_of(x, rest) == b) take(x, s.list[i], rest);
        }
      } else {
        find.scan_row({b, b}, kNoBins, [&](uint64_t at, double rs) { take(logit_of(at), at, rs); });
      }
      if (mine) atomicAdd(reinterpret_cast<unsigned long long*>(t.weight), (unsigned long long)mine);
      __syncthreads();
      total = least_of(total, within(b, t.weight[0]));
      if (b < cut) cut = b, cut_at = ~0ull;
    }
  }
  // ---- the token
  const double target = u * (double)total;
  const int b = min(find.find_bin(kPasses, target), cut);
  uint64_t sum, at = find.resolve(b, kPasses, (target - (double)before(b)) / scale_of(b), sum);
  if (b == cut && at > cut_at) at = cut_at;
  if (tid == 0) {
    const double log2_total = log2((double)total) - kPoint;
    const double n_at = grid(logit_of(at), c, rest);
    a.tokens[row] = (int64_t)(uint32_t)at;
    a.logprobs[row] = (float)((((n_at - ref) + rest) / 16 - log2_total) * 0.6931471805599453);
    if (a.rows) a.rows[row] = RowState{c, ref, low, log2_total, cut_at, cut, 0};
  }
}

// --------------------------------------------------------- probabilities

constexpr int PT = 256, PIECES = 4;

template <typename T>
__global__ __launch_bounds__(PT) void sample_probs(SampleArgs a, int blocks) {
  const int row = (int)(blockIdx.x / (uint32_t)blocks), block = (int)(blockIdx.x - (uint32_t)row * blocks);
  const RowReader<T> r(a, row);
  const RowState s = a.rows[row];
  float* out = a.probs + (int64_t)row * a.ld_probs;
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const int piece = (block * PIECES + j) * PT + threadIdx.x, i0 = r.first(piece);
    const u32x4 w = r.load(piece);
    float p[RowReader<T>::W];
#pragma unroll
    for (int e = 0; e < RowReader<T>::W; ++e) {
      const float x = finite_top(r.at(w, e));
      double rest;
      const double n = grid(x, s.c, rest), d = s.ref - n;
      p[e] = 0.f;
      if (s.cut >= 0 && d <= s.cut && (double)x * s.c >= s.low && (d < s.cut || place(x, i0 + e) <= s.cut_at)) {
        // 2^whole 2^part: the exponential sees a small number
        const double y = (rest - d) / 16 - s.log2_total, whole = rint(y);
        p[e] = ldexpf(__builtin_amdgcn_exp2f((float)(y - whole)), (int)whole);
      }
      if (s.cut == kOneHot) p[e] = i0 + e == s.token ? 1.f : 0.f;
      if (s.cut == kNone) p[e] = __builtin_nanf("");
    }
#pragma unroll
    for (int e = 0; e < RowReader<T>::W; ++e)
      if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = p[e];
  }
}

// ------------------------------------------------------------------ host

// Chunks of 16384 logits where they fill the CUs, else of 4096.
struct Plan {
  int64_t chunk, chunks;
  int64_t heads, weights, counts, rows;  // bytes
  int64_t bytes() const { return heads + weights + counts + rows; }
};

Plan plan_of(int64_t B, int64_t V, bool counted, bool probs) {
  Plan p;
  p.chunk = B * ((V + 16383) / 16384) >= 1024 ? 16384 : 4096;
  p.chunks = (V + 7 + p.chunk - 1) / p.chunk;  // 7: a row may begin inside its first piece
  p.heads = B * p.chunks * (int64_t)sizeof(ChunkHead);
  p.weights = B * p.chunks * kBins * 8;
  p.counts = counted ? B * p.chunks * kBins * 4 : 0;
  p.rows = probs ? B * (int64_t)sizeof(RowState) : 0;
  return p;
}

template <typename T>
int32_t launch(const SampleArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((uint32_t)(a.B * p.chunks));
  if (p.chunk == 16384)
    sample_chunks<T, 32><<<grid, dim3(CT), 0, st>>>(a);
  else
    sample_chunks<T, 8><<<grid, dim3(CT), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  static bool done[kDevices] = {};
  const int32_t r = allow_lds(reinterpret_cast<const void*>(&sample_rows<T>), sizeof(RowLds), done);
  if (r != CATOPT_OK) return r;
  sample_rows<T><<<dim3((uint32_t)a.B), dim3(RT), sizeof(RowLds), st>>>(a);
  CATOPT_LAUNCH_CHECK();
  if (a.probs) {
    constexpr int64_t per = PT * PIECES * RowReader<T>::W;
    const int64_t blocks = (a.V + RowReader<T>::W - 1 + per - 1) / per;
    sample_probs<T><<<dim3((uint32_t)(a.B * blocks)), dim3(PT), 0, st>>>(a, (int)blocks);
    CATOPT_LAUNCH_CHECK();
  }
  return CATOPT_OK;
}

bool overlaps(const void* p, int64_t n, const void* q, int64_t m) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return p && q && n > 0 && m > 0 && a < b + (uintptr_t)m && b < a + (uintptr_t)n;
}

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int64_t catopt_hip_sample_workspace_bytes(int64_t B, int64_t V, int32_t counted, int32_t probs) {
  if (B < 0 || V < 1 || V > kMaxVocab || B > (1 << 20)) return -1;
  if (B * V >= (1LL << 36)) return -1;
  return plan_of(B, V, counted != 0, probs != 0).bytes();
}

extern "C" int32_t catopt_hip_sample(int32_t dtype, int64_t B, int64_t V, const void* logits, int64_t ld, const float* u,
                                     const float* temperature, double temperature_all, const int32_t* top_k,
                                     int64_t top_k_all, const float* top_p, double top_p_all, const float* min_p,
                                     double min_p_all, int64_t* tokens, float* logprobs, float* probs, int64_t ld_probs,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  if (B < 0 || V < 1) return CATOPT_E_INVAL;
  if (dtype != CATOPT_F32 && dtype != CATOPT_BF16) return CATOPT_E_UNSUPPORTED;
  const bool counted = top_k || top_k_all > 1;
  const int64_t need = catopt_hip_sample_workspace_bytes(B, V, counted, probs != nullptr);
  if (need < 0) return CATOPT_E_UNSUPPORTED;
  if (B == 0) return CATOPT_OK;
  if (!logits || !u || !tokens || !logprobs || ld < 0 || (B > 1 && ld_probs < V && probs)) return CATOPT_E_INVAL;
  const int64_t size = dtype == CATOPT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return CATOPT_E_INVAL;
  const struct {
    const void* p;
    int64_t n;
  } out[3] = {{tokens, 8 * B}, {logprobs, 4 * B}, {probs, 4 * ((B - 1) * ld_probs + V)}},
    in[6] = {{logits, size * ((B - 1) * ld + V)}, {u, 4 * B}, {temperature, 4 * B}, {top_k, 4 * B}, {top_p, 4 * B}, {min_p, 4 * B}};
  for (int i = 0; i < 3; ++i) {
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i].p, out[i].n, out[j].p, out[j].n)) return CATOPT_E_INVAL;
    for (const auto& x : in)
      if (overlaps(out[i].p, out[i].n, x.p, x.n)) return CATOPT_E_INVAL;
  }
  if (!workspace || workspace_bytes < need || !aligned16(workspace)) return CATOPT_E_WORKSPACE;
  const Plan p = plan_of(B, V, counted, probs != nullptr);
  if (!grid_fits(B * p.chunks, CT) || !grid_fits(B, RT) || !grid_fits(B * ((V + 4095) / 4096 + 1), PT)) return CATOPT_E_UNSUPPORTED;
  SampleArgs a{};
  a.x = logits, a.ld = B > 1 ? ld : 0, a.ld_probs = B > 1 ? ld_probs : 0, a.V = (int)V, a.B = (int)B, a.chunks = (int)p.chunks;
  a.t_row = temperature, a.p_row = top_p, a.low_row = min_p, a.k_row = top_k;
  a.t = temperature_all, a.p = top_p_all, a.low = min_p_all, a.k = top_k_all;
  a.u = u, a.tokens = tokens, a.logprobs = logprobs, a.probs = probs;
  char* ws = static_cast<char*>(workspace);
  a.rows = probs ? reinterpret_cast<RowState*>(ws) : nullptr;
  ws += p.rows;
  a.weights = reinterpret_cast<uint64_t*>(ws);
  ws += p.weights;
  a.heads = reinterpret_cast<ChunkHead*>(ws);
  ws += p.heads;
  a.counts = reinterpret_cast<uint32_t*>(ws);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CATOPT_F32 ? launch<float>(a, p, st) : launch<uint16_t>(a, p, st);
}
