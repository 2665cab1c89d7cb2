// What follows the attention kernels: the combination of split keys' carriers,
// and the keys' weights where the few-row kernel has stored its products (4
// bytes a row and key, against 4 d bytes for K and V).  A call that needs both
// takes one launch: the weights' workgroups work out the rows' statistics from
// the ranges' themselves instead of waiting for the combination.  Both are
// latency: 4.8 us for a step of 32 sequences, 6.6 with the weights of 47000 keys.
#include "paged_attn.hpp"

namespace catopt {
namespace {

constexpr int NT = 256;

// WAVES waves per row (token, query head): the carriers of its key ranges, D / 4
// lanes to a range's numerators, so that 2 WAVES (D = 64: 4 WAVES) ranges load
// at once.  R: the rows of the tiles they were made with.
template <int D, int R, int WAVES>
__device__ __forceinline__ void combine_rows(const PagedArgs& a, int block) {
  constexpr int TPR = D / 4, GROUPS = 64 * WAVES / TPR;
  const int lane = threadIdx.x & 63, tid = WAVES == 4 ? threadIdx.x : lane;
  const int row = WAVES == 4 ? block : block * 4 + (int)(threadIdx.x >> 6);  // N Hq < 2^30
  if (row >= a.N * a.Hq) return;
  const int n = (int)a.q_heads.div(row), hq = row - n * a.Hq;
  int b = -1;
  for (int c0 = 0; c0 < a.B; c0 += 64) {  // the last sequence that starts at or before the token
    const int i = c0 + lane;
    const int k = __popcll(__ballot(i < a.B && min(max(a.starts[i < a.B ? i : 0], 0), (int)a.N) <= n));
    b += k;
    if (k < 64) break;
  }
  if (b < 0) return;
  PagedTile x{};
  x.b = b;
  seq_rows(a.starts, b, a.N, x.row0, x.nq);
  if (n < x.row0 || n >= x.row0 + x.nq) return;
  x.len = min(max(a.lens[b], 0), a.cap);
  x.r0 = ((n - x.row0) * a.G + hq - (int)a.group.div(hq) * a.G) / R * R;
  x.rows = min(R, x.nq * a.G - x.r0);
  paged_ranges(a, x);
  if (!x.split) return;  // written by the tile
  const int splits = count_ranges(x);
  const float c = a.scale * kLog2e;
  const float* ml = a.part + (int64_t)2 * row * a.splits;
  const float* num =
      a.part + ((2 * a.N * a.Hq * a.splits + 3) & ~(int64_t)3) + (int64_t)row * a.splits * D + 4 * (tid % TPR);
  // lane s of every wave: range s (64 at most)
  const bool mine = lane < splits;
  const float ms = mine ? ml[2 * lane] : kNegInf, ls = mine ? ml[2 * lane + 1] : 0.f;
  float mx = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  const float f = mine ? move_factor(ms, mx, c) : 0.f;
  float lt = ls * f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) lt += __shfl_xor(lt, o, 64);
  f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 8;  // loads ahead of their additions
  for (int s0 = 0; s0 < splits; s0 += U * GROUPS) {  // every lane stays: the factors come from lanes
    f32x4 ys[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + i * GROUPS + tid / TPR;
      ys[i] = s < splits ? *reinterpret_cast<const f32x4*>(num + (int64_t)s * D) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < U; ++i) y += ys[i] * __shfl(f, min(s0 + i * GROUPS + tid / TPR, 63), 64);
  }
  if constexpr (WAVES == 4) {
    __shared__ f32x4 sums[GROUPS][TPR];
    sums[tid / TPR][tid % TPR] = y;
    __syncthreads();
    if (tid < TPR) {
#pragma unroll
      for (int i = 1; i < GROUPS; ++i) y += sums[i][tid];
    }
  } else {
#pragma unroll
    for (int o = TPR; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], o, 64);
  }
  if (tid < TPR && 4 * tid < a.d) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = finish(y[e], lt, a.normalize);
    *reinterpret_cast<u32x2*>(a.o + (int64_t)n * a.o_t + (int64_t)hq * a.o_h + 4 * tid) =
        u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  }
  if (tid == 0) row_stats(a, row, mx, lt);
}

// The row_log of row i, all lanes of a wave together, from its ranges' carriers.
__device__ __forceinline__ float ranges_log(const PagedArgs& a, int64_t i, int splits) {
  const int lane = threadIdx.x & 63;
  const float* ml = a.part + 2 * i * a.splits;
  const bool mine = lane < splits;
  const float c = a.scale * kLog2e, m = mine ? ml[2 * lane] : kNegInf, l = mine ? ml[2 * lane + 1] : 0.f;
  float mx = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  float lt = mine ? l * move_factor(m, mx, c) : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) lt += __shfl_xor(lt, o, 64);
  return lt == 0.f ? __builtin_inff() : mx * c + __builtin_amdgcn_logf(lt);
}

constexpr int kLogRows = 64;  // rows whose statistics are in LDS at a time

// Four keys per thread: their stored products of every row that sees them.
__device__ __forceinline__ void weights_of_scores(const PagedArgs& a, int block, int blocks) {
  __shared__ float logs[kLogRows];
  const int bh = block / blocks, b = (int)a.k_heads.div(bh), h = bh - b * a.Hkv, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int key0 = (block - bh * blocks) * NT * 4, key = key0 + 4 * threadIdx.x;
  PagedTile x{};
  x.b = b;
  seq_rows(a.starts, b, a.N, x.row0, x.nq);
  x.len = min(max(a.lens[b], 0), a.cap);
  if (key0 >= x.len) return;
  const int old = x.len - x.nq, rows = x.nq * a.G;
  const float c = a.scale * kLog2e;
  // the page of the four keys; of an invalid one they count as masked, whatever the
  // rows hold (a NaN would pass their stored -inf)
  const int page = group_page(a, a.table + (int64_t)b * a.table_ld, key, x.len);
  f32x4 w = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < rows; r0 += kLogRows) {
    const int n = min(rows - r0, kLogRows);
    __syncthreads();  // the rows before have been used
    for (int r = wave; r < n; r += NT / 64) {
      const int tok = (int)a.group.div(r0 + r);
      const int64_t i = (int64_t)(x.row0 + tok) * a.Hq + h * a.G + r0 + r - tok * a.G;
      x.r0 = (r0 + r) / kFewRows * kFewRows;
      x.rows = min(kFewRows, rows - x.r0);
      paged_ranges(a, x);
      const float o = x.split ? ranges_log(a, i, count_ranges(x)) : a.row_log[i];
      if (lane == 0) logs[r] = o;
    }
    __syncthreads();
    for (int r = 0; r < n; ++r) {
      const int tok = (int)a.group.div(r0 + r), seen = a.causal ? old + tok : x.len - 1;  // last key
      if (key > seen) continue;
      const int64_t i = (int64_t)(x.row0 + tok) * a.Hq + h * a.G + r0 + r - tok * a.G;
      const f32x4 s = *reinterpret_cast<const f32x4*>(a.scores + i * a.cap + key);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -logs[r]));
        w[e] += key + e <= seen ? y : 0.f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (key + e < x.len) add_weight(a, b, h, key + e, old, page >= 0 && page < a.n_pages ? w[e] : 0.f);
}

template <int D, int R, int WAVES>
__global__ __launch_bounds__(NT) void paged_combine(PagedArgs a) {
  combine_rows<D, R, WAVES>(a, blockIdx.x);
}

__global__ __launch_bounds__(NT) void paged_score_weights(PagedArgs a, int blocks) {
  weights_of_scores(a, blockIdx.x, blocks);
}

// The weights' workgroups first: they are the longer ones.
template <int D, int WAVES>
__global__ __launch_bounds__(NT) void paged_combine_and_weights(PagedArgs a, int blocks, int weight_blocks) {
  if ((int)blockIdx.x < weight_blocks)
    weights_of_scores(a, blockIdx.x, blocks);
  else
    combine_rows<D, kFewRows, WAVES>(a, blockIdx.x - weight_blocks);
}

template <int D>
int32_t finish_launch(const PagedArgs& a, bool few, hipStream_t s) {
  // four waves a row where the rows alone do not fill the CUs
  const int64_t rows = a.N * a.Hq;
  const bool wide = rows < 2048;
  const int64_t nc = wide ? rows : (rows + 3) / 4;
  const int64_t blocks = (a.cap + 4 * NT - 1) / (4 * NT), nw = a.scores ? (int64_t)a.B * a.Hkv * blocks : 0;
  if (!grid_fits(nc + nw, NT)) return CATOPT_E_UNSUPPORTED;
  const dim3 grid((uint32_t)(nc + nw)), threads(NT);
  if (a.scores) {
    if (wide)
      paged_combine_and_weights<D, 4><<<grid, threads, 0, s>>>(a, (int)blocks, (int)nw);
    else
      paged_combine_and_weights<D, 1><<<grid, threads, 0, s>>>(a, (int)blocks, (int)nw);
  } else if (few) {
    if (wide)
      paged_combine<D, kFewRows, 4><<<grid, threads, 0, s>>>(a);
    else
      paged_combine<D, kFewRows, 1><<<grid, threads, 0, s>>>(a);
  } else {
    if (wide)
      paged_combine<D, kTileRows, 4><<<grid, threads, 0, s>>>(a);
    else
      paged_combine<D, kTileRows, 1><<<grid, threads, 0, s>>>(a);
  }
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_finish_launch(const PagedArgs& a, int D, bool few, hipStream_t s) {
  return D == 128 ? finish_launch<128>(a, few, s) : finish_launch<64>(a, few, s);
}

int32_t paged_score_weights_launch(const PagedArgs& a, hipStream_t s) {
  const int64_t blocks = (a.cap + 4 * NT - 1) / (4 * NT), n = (int64_t)a.B * a.Hkv * blocks;
  if (!grid_fits(n, NT)) return CATOPT_E_UNSUPPORTED;
  paged_score_weights<<<dim3((uint32_t)n), dim3(NT), 0, s>>>(a, (int)blocks);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace catopt
