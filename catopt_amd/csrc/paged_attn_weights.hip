// Every cached key's attention weight, summed over the new tokens and the
// query heads of its key head:
//   w[j] = sum_rows exp(s_rj - m_r) / l_r = sum_rows exp2(q_r . k_j c - o_r),
//   c = scale log2 e,  o_r = m_r log2 e + log2 l_r  (PagedArgs::row_log)
// on top of the weight so far (nothing for the new tokens' own keys).
//
// This is the form for many rows (with few, the attention kernel stores its
// products): they are formed again, half of the attention's work.  A workgroup
// keeps 128 keys in registers, 32 per wave, and streams the rows by 32 through
// LDS; the score accumulator's columns are rows, so each lane adds its rows for
// 16 keys and the lanes meet once at the end.  Each product's scores take an
// exponential, a multiply-add and an addition, which costs more than the MFMA, so
// the rows' addresses and offsets are kept to a few additions a step.  64 keys a
// wave (half the LDS reads, two waves to a SIMD instead of four) took 200 us where
// this took 168, now 164: 2048 tokens over 8192 keys, 32 query heads on 8, 730
// TFLOP/s.  There VALU and MFMA fill the SIMDs (0.55 and 0.35 of the cycles).  Two
// chunks of 700 and 1100 tokens over 2200 and 4600 keys take 81 us with 0.43 and
// 0.26: 1296 workgroups of 1 to 46 steps on 1024 places.  Where the keys leave
// CUs idle the rows are split over workgroups and the parts added in order by
// another launch.
#include "paged_attn.hpp"

namespace catopt {
namespace {

constexpr int NT = 256;

constexpr int kKeys = 128;  // of a workgroup, 32 per wave

template <int D>
__global__ __launch_bounds__(NT, 2) void weights_of_rows(PagedArgs a, FastDiv blocks, FastDiv parts, float* part) {
  // rows a 16-byte piece further apart than they are long: 16 rows' pieces lie
  // in different banks, and a fragment's address is one register and a constant
  constexpr int ROW = D * 2 + 16;
  __shared__ __attribute__((aligned(16))) char lds[2][32 * ROW];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t hs = a.k_heads.div(blockIdx.x), ps = parts.div(hs);
  const int h = (int)(blockIdx.x - hs * a.k_heads.d), pt = (int)(hs - ps * parts.d);
  const int b = (int)blocks.div(ps), blk = (int)(ps - (uint32_t)b * blocks.d);
  int row0, nq;
  seq_rows(a.starts, b, a.N, row0, nq);
  const int len = min(max(a.lens[b], 0), a.cap);
  if (blk * kKeys >= len) return;
  const int old = len - nq, off = a.causal ? old : 0x3fffffff;
  const int key0 = blk * kKeys + 32 * wave;
  const float c = a.scale * kLog2e;

  bf16x8 kf[D / 16];
  uint64_t ok;  // keys whose page is one
  {
    const int key = key0 + l32;
    bool valid = key < len;
    const uint32_t tp = a.page.div(valid ? key : 0);
    const int64_t page = valid ? a.table[(int64_t)b * a.table_ld + tp] : -1;
    valid = page >= 0 && page < a.n_pages;
    const uint16_t* k = a.k + (valid ? page * a.k_p + h * a.k_h + (int64_t)(key - (int)(tp * a.page.d)) * a.k_s : 0);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      u32x4 w = u32x4{0, 0, 0, 0};
      if (valid && 16 * j + 8 * g < a.d) w = *reinterpret_cast<const u32x4*>(k + 16 * j + 8 * g);
      kf[j] = __builtin_bit_cast(bf16x8, w);
    }
    ok = __ballot(valid);
  }

  // steps of 32 rows from the first that sees the block's first key; this part's share
  const int rows = nq * a.G, tok0 = max(blk * kKeys - off, 0);
  const int ta = (int)min((int64_t)tok0 * a.G, (int64_t)rows) / 32, tb = (rows + 31) / 32;
  const int t0 = ta + (int)parts.div((tb - ta) * pt), t1 = ta + (int)parts.div((tb - ta) * (pt + 1));  // below 2^30

  constexpr int CH = AttnRow<D>::CH, LD = 32 * CH / NT;  // 16-byte pieces of a step per thread
  static_assert(LD >= 1 && LD <= 2, "the pieces' registers");
  u32x4 qr[2];
  float o_next = 0.f;
  // Row r of the sequence is token r / G, head r % G.  The rows that a lane
  // reads advance by 32 a step, so their tokens and heads, and with them the
  // offsets of their queries and offsets o, advance by constants and a carry.
  struct Walk {
    int r, g;
    int64_t q, o;
  };
  const int step_t = 32 / a.G, step_g = 32 - step_t * a.G;
  const int64_t step_q = step_t * a.q_t + step_g * a.q_h, wrap_q = a.q_t - a.G * a.q_h;
  const int64_t step_o = (int64_t)step_t * a.Hq + step_g, wrap_o = a.Hq - a.G;
  auto walk_from = [&](int r) {
    const int tok = (int)a.group.div(r), gr = r - tok * a.G;
    return Walk{r, gr, (int64_t)(row0 + tok) * a.q_t + (int64_t)(h * a.G + gr) * a.q_h,
                (int64_t)(row0 + tok) * a.Hq + h * a.G + gr};
  };
  auto advance = [&](Walk& x, bool queries) {
    x.r += 32;
    if (queries)
      x.q += step_q;
    else
      x.o += step_o;
    if (step_g == 0) return;  // G divides 32: the heads stay
    x.g += step_g;
    const bool wrap = x.g >= a.G;
    x.g -= wrap ? a.G : 0;
    if (queries)
      x.q += wrap ? wrap_q : 0;
    else
      x.o += wrap ? wrap_o : 0;
  };
  Walk wq[2];
#pragma unroll
  for (int i = 0; i < LD; ++i) {
    wq[i] = walk_from(32 * t0 + (i * NT + tid) / CH);
    wq[i].q += (tid % CH) * 8;
  }
  Walk wo = walk_from(32 * t0 + l32);
  const bool column = (tid % CH) * 8 < a.d;
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      qr[i] = u32x4{0, 0, 0, 0};
      if (wq[i].r < rows && column) qr[i] = *reinterpret_cast<const u32x4*>(a.q + wq[i].q);
      advance(wq[i], true);
    }
    o_next = wo.r < rows ? a.row_log[wo.o] : __builtin_inff();
    advance(wo, false);
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int piece = i * NT + tid;
      *reinterpret_cast<u32x4*>(lds[buf] + piece / CH * ROW + piece % CH * 16) = qr[i];
    }
  };

  float w[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) w[r] = 0.f;
  if (t0 < t1) {
    fetch();
    stage(0);
  }
  auto step = [&](int t, int buf) {
    const float o = o_next;
    __syncthreads();  // the step is staged, and the other buffer is free
    if (t + 1 < t1) fetch();
    const int first = off + (int)a.group.div(32 * t);                     // last key of the step's first row
    const int last = off + (int)a.group.div(min(32 * t + 32, rows) - 1);  // and of its last row
    if (key0 <= last && key0 < len) {
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        s = mfma32x32x16(kf[j], *reinterpret_cast<const bf16x8*>(lds[buf] + l32 * ROW + (2 * j + g) * 16), s);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, -o);
      // The mask is for the exponents: a row whose o is NaN adds nothing to keys that
      // it does not see.  One behind the last (staged as zeros) sees none: against an
      // infinite key its score is NaN.
      if (key0 + 31 > first || 32 * t + 32 > rows) {
        const int lim = 32 * t + l32 < rows ? off + (int)a.group.div(32 * t + l32) : -1;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = key0 + acc_row(r, g) <= lim ? s[r] : kNegInf;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] += __builtin_amdgcn_exp2f(s[r]);
    }
    if (t + 1 < t1) stage(buf ^ 1);
  };
  for (int t = t0; t < t1; t += 2) {  // in pairs: the buffer is a constant of the addresses
    step(t, 0);
    if (t + 1 < t1) step(t + 1, 1);
  }
  // The halves' 32 lanes meet: in each step a lane hands half of its keys' sums to
  // the lane whose index differs in one bit and takes that one's of the others, so
  // that two neighbours end with the key of register l32 / 2.  16 exchanges, where
  // summing each key over all lanes takes 80.
#pragma unroll
  for (int x = 16, n = 8; n > 0; x >>= 1, n >>= 1) {
    const bool upper = l32 & x;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? w[i + n] : w[i], give = upper ? w[i] : w[i + n];
      w[i] = keep + __shfl_xor(give, x, 64);
    }
  }
  w[0] += __shfl_xor(w[0], 1, 64);
  const int in = 8 * (l32 >> 3) + 4 * g + ((l32 >> 1) & 3), j = key0 + in;  // acc_row(l32 / 2, g)
  if (l32 & 1 || j >= len) return;
  const float y = (ok >> in) & 1 ? w[0] : 0.f;
  if (parts.d > 1)
    part[((int64_t)(pt * a.B + b) * a.Hkv + h) * a.cap + j] = y;
  else
    add_weight(a, b, h, j, old, y);
}

__global__ __launch_bounds__(NT) void weights_add_parts(PagedArgs a, int blocks, int parts, const float* part) {
  const int bh = blockIdx.x / blocks, b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int key = (blockIdx.x - bh * blocks) * NT + threadIdx.x;
  int row0, nq;
  seq_rows(a.starts, b, a.N, row0, nq);
  const int len = min(max(a.lens[b], 0), a.cap);
  if (key >= len) return;
  float w = 0.f;
  for (int p = 0; p < parts; ++p) w += part[((int64_t)p * a.B * a.Hkv + bh) * a.cap + key];
  add_weight(a, b, h, key, len - nq, w);
}

}  // namespace

// Parts of the rows: as many as give eight workgroups to a CU, were every
// sequence as long as its table.
int paged_weight_parts(int64_t B, int64_t Hkv, int64_t cap, int64_t N, int64_t G) {
  const int64_t groups = B * Hkv * ((cap + kKeys - 1) / kKeys);
  int64_t n = groups > 0 ? 2048 / groups : 1;
  const int64_t steps = N * G / 32;
  if (n > steps / 8) n = steps / 8;  // of the call: a part has a few steps at least
  return n < 1 ? 1 : n > 16 ? 16 : (int)n;
}

int32_t paged_weights_launch(const PagedArgs& a, int D, int parts, float* part, hipStream_t s) {
  if (a.cap == 0) return CATOPT_OK;
  const int64_t heads = (int64_t)a.B * a.Hkv;
  if (a.scores) return paged_score_weights_launch(a, s);
  const int64_t blocks = (a.cap + kKeys - 1) / kKeys;
  if (!grid_fits(heads * blocks * parts, NT)) return CATOPT_E_UNSUPPORTED;
  const dim3 grid((uint32_t)(heads * blocks * parts));
  if (D == 128)
    weights_of_rows<128><<<grid, dim3(NT), 0, s>>>(a, FastDiv::of(blocks), FastDiv::of(parts), part);
  else
    weights_of_rows<64><<<grid, dim3(NT), 0, s>>>(a, FastDiv::of(blocks), FastDiv::of(parts), part);
  CATOPT_LAUNCH_CHECK();
  if (parts > 1) {
    const int64_t n = (a.cap + NT - 1) / NT;
    if (!grid_fits(heads * n, NT)) return CATOPT_E_UNSUPPORTED;
    weights_add_parts<<<dim3((uint32_t)(heads * n)), dim3(NT), 0, s>>>(a, (int)n, parts, part);
    CATOPT_LAUNCH_CHECK();
  }
  return CATOPT_OK;
}

}  // namespace catopt
