// Paged attention with few query rows per key head (a generation step: one
// token of each sequence, its G query heads sharing a key head).
//
// K and V are read once and used by at most 32 rows, so HBM bounds it.  A
// workgroup takes a range of the keys of one tile of 32 rows and one key head;
// its waves take 32 keys each of every stage, and the ranges' carriers (m, l,
// numerator) are combined by a second launch where there are several.
//
// Products as in the contiguous kernels: S^T = K Q^T and O^T += V^T P^T on the
// 32x32x16 MFMA, the accumulator column the query row.  A wave's rows of K and
// V go global->LDS directly into two stages of its own.  A stage is loaded again
// as soon as it has been used, and the wait for the other one leaves the new
// loads in flight: the waves read nothing of each other's, so there is no
// barrier in the loop.  The loads carry the non-temporal hint: a step of 32
// sequences over 131072 keys 115 -> 101 us with the combination, 536 MB and so 5.3
// TB/s; a step over 47000 keys with their weights 55 -> 49.  A lane works out the
// place of 8 keys, the wave those of 16 stages at once.
//
// The softmax terms are summed in fp32 and rounded to bf16 for the product with V,
// as in the 128-row kernel, so that both are as exact whichever of them a call takes:
// off by 0.0021 to 0.0022 of the result's size on random inputs, where the result's
// own rounding gives 0.0017.
#include "paged_attn.hpp"

namespace catopt {
namespace {

// Two waves (D = 64: four) of two stages fill at most half a CU's LDS, so that
// two workgroups share it and one's start runs under the other's loads: the form
// for long keys.  Four waves at D = 128 took 182 us for the step above.  Eight
// waves of one stage (WIDE) have 256 keys in flight at once: the form for one
// range of few keys, which spares the second launch.
template <int D, bool WIDE>
struct Few {
  static constexpr int WAVES = WIDE ? 8 : D == 128 ? 2 : 4, NT = 64 * WAVES, STAGES = WIDE ? 1 : 2;
  static constexpr int KEYS = 32 * WAVES;              // of a round of stages, 32 per wave
  static constexpr int HALF = 32 * AttnRow<D>::BYTES;  // a wave's K (or V) rows of a stage
  static constexpr int STAGE = 2 * HALF, WAVE_BYTES = STAGES * STAGE;
  static constexpr int LOADS = HALF / 1024;            // 1 KB loads of K (and of V) per stage
  static constexpr int ROWS = 32 / LOADS;              // rows of one
  static constexpr int OLD = D + 4;                    // row of the merge buffer, floats
  static constexpr int LOOP = WAVES * WAVE_BYTES, MERGE = WAVES * 32 * OLD * 4 + WAVES * 64 * 4;
  static constexpr int BYTES = LOOP > MERGE ? LOOP : MERGE;  // the merge reuses the stages
};

// Wait for all but the newest LOADS * 2 loads (one stage's), or for all.  The
// stage waited for is older than those whatever else the compiler has issued in
// between, and the asm keeps the stage's LDS reads behind it.
template <int N>
__device__ __forceinline__ void wait_stage(bool newer) {
  if (newer)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int D, bool WIDE>
__global__ __launch_bounds__((Few<D, WIDE>::NT), 2) void paged_few_kernel(PagedArgs a) {
  using L = Few<D, WIDE>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int h, t, split;
  decode_block(a, h, t, split);
  PagedTile x = paged_tile<kFewRows>(a, t);
  if (x.rows == 0) return;
  paged_ranges(a, x);
  if (!has_range(x, split)) return;
  const float c = a.scale * kLog2e;

  // this wave's stages: 32 keys each from key_of(i) on
  const int k_begin = split * x.keys + 32 * wave, k_end = min(x.kend, (split + 1) * x.keys);
  const int stages = k_end > k_begin ? (k_end - k_begin + L::KEYS - 1) / L::KEYS : 0;
  auto key_of = [&](int i) { return k_begin + i * L::KEYS; };
  const int32_t* table = a.table + (int64_t)x.b * a.table_ld;
  const uint16_t *kb = a.k + (int64_t)h * a.k_h, *vb = a.v + (int64_t)h * a.v_h;
  // the page of this lane's 8 keys of the 16 stages from stage st on; the first
  // ones on their way before the queries are
  auto lane_key = [&](int st) { return key_of(st + (lane >> 2)) + 8 * (lane & 3); };
  const int first_page = group_page(a, table, lane_key(0), lane_key(0) < k_end ? x.len : 0);

  // this lane's query row
  const int row = x.r0 + l32, tok = (int)a.group.div(row), hq = h * a.G + row - tok * a.G;
  const bool live = l32 < x.rows;
  const uint16_t* q = a.q + (int64_t)(x.row0 + tok) * a.q_t + (int64_t)hq * a.q_h;
  bf16x8 qf[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    u32x4 w = u32x4{0, 0, 0, 0};
    if (live && 16 * j + 8 * g < a.d) w = *reinterpret_cast<const u32x4*>(q + 16 * j + 8 * g);
    qf[j] = __builtin_bit_cast(bf16x8, w);
  }
  const int lim = min(x.off + tok, x.len - 1);  // last key this row sees
  const int lim0 = x.off + (int)a.group.div(x.r0);  // and the tile's first

  // a lane's 16 bytes of load k: row k ROWS + lane / CH of the stage, row & 7 of
  // its group; the swizzles depend on a row's place among 16 (K, D = 128: loads
  // k and k + 4 agree), 8 or 4 rows
  const int sub = lane / AttnRow<D>::CH, cp = lane % AttnRow<D>::CH;
  uint32_t koff[4], voff[2];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = k * L::ROWS + sub;
    koff[k] = group_offset(a.k_s, r & 7, cp ^ (r & (AttnRow<D>::CH - 1) & 15), a.d);
    if (k < 2) voff[k] = group_offset(a.v_s, r & 7, cp ^ vswz<D>(r), a.d);
  }
  const uint32_t lds0 = lds_u32(lds) + wave * L::WAVE_BYTES;
  auto issue = [&](int i, int lane0, const KeyGroup& at) {  // stage i, its groups in lanes lane0 to lane0 + 3
#pragma unroll
    for (int k = 0; k < L::LOADS; ++k) {
      const int ln = lane0 + k * L::ROWS / 8;
      const uint32_t to = lds0 + (i & (L::STAGES - 1)) * L::STAGE + k * 1024;
      dma_rows_once(k_rsrc(at, ln), koff[k & 3], v_rsrc(at, ln), voff[k & 1], to, L::HALF);
    }
  };

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m = kNegInf, l = 0.f;
  float* srow = a.scores ? a.scores + ((int64_t)(x.row0 + tok) * a.Hq + hq) * a.cap : nullptr;

#pragma unroll
  for (int j = 0; j < D / 16; ++j)  // the queries have arrived: no wait for them below, which would wait for K and V
    asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[j])));

  KeyGroup at;
  uint64_t bad;
  auto places = [&](int st, int page) {
    bool odd;
    at = key_group(a, kb, vb, page, lane_key(st), lane_key(st) < k_end ? x.len : 0, odd);
    bad = __ballot(odd);
  };
  places(0, first_page);
  for (int st = 0; st < stages; ++st) {
    const int in = st & 15;  // of the 16 stages whose groups the lanes hold
    if (in == 0 && st > 0) places(st, group_page(a, table, lane_key(st), lane_key(st) < k_end ? x.len : 0));
    if (in == 0 || L::STAGES == 1) issue(st, 4 * in, at);
    const bool newer = L::STAGES == 2 && in < 15 && st + 1 < stages;
    if (newer) issue(st + 1, 4 * in + 4, at);
    wait_stage<2 * L::LOADS>(newer);
    const int key0 = key_of(st);
    const uint32_t bad_now = (uint32_t)(bad >> (4 * in)) & 15u;
    const char* Ks = lds + wave * L::WAVE_BYTES + (st & (L::STAGES - 1)) * L::STAGE;
    const char* Vs = Ks + L::HALF;

    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      s = mfma32x32x16(*reinterpret_cast<const bf16x8*>(Ks + tile_off<D>(l32, 2 * j + g)), qf[j], s);
    // some row does not see some key: the first row sees the fewest
    const bool masked = key0 + 32 > x.len || key0 + 31 > lim0 || bad_now;
    if (masked) mask_scores(s, lim - key0, bad_now);
    if (srow && live) {
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int key = key0 + 8 * rg + 4 * g;  // cap is a multiple of 8
        if (key < a.cap)
          *reinterpret_cast<f32x4*>(srow + key) = f32x4{s[4 * rg], s[4 * rg + 1], s[4 * rg + 2], s[4 * rg + 3]};
      }
    }
    float mt = kNegInf;
#pragma unroll
    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[r]);
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float m_new = fmaxf(m, mt);
    const float alpha = move_factor(m, m_new, c);
    m = m_new;
    const float mr = m == kNegInf ? 0.f : m;
    float lsum = 0.f;
    bf16x8 p[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -mr * c));
      lsum += e;
      p[r >> 3][r & 7] = static_cast<__bf16>(e);
    }
    l = l * alpha + lsum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
    }
    bf16x8 vf[D / 16];
    read_v<D>(Vs, 0, vf);
    if (masked && odd_values<D>(vf)) take_odd_values<D>(vf, lim - key0, bad_now, acc);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[db] = mfma32x32x16(vf[2 * db + u], p[u], acc[db]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this stage's LDS reads are done: it may be loaded again
  }

  // ---- the waves' carriers meet in LDS: [wave][row][d] numerators, then
  // [wave][row] (m, l)
  __syncthreads();  // every wave is done with the stages
  l += __shfl_xor(l, 32, 64);
  float* num = reinterpret_cast<float*>(lds);
  float* ml = num + L::WAVES * 32 * L::OLD;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg)
      *reinterpret_cast<f32x4*>(num + (wave * 32 + l32) * L::OLD + 32 * db + 8 * rg + 4 * g) =
          f32x4{acc[db][4 * rg], acc[db][4 * rg + 1], acc[db][4 * rg + 2], acc[db][4 * rg + 3]};
  if (g == 0) {
    ml[(wave * 32 + l32) * 2] = m;
    ml[(wave * 32 + l32) * 2 + 1] = l;
  }
  __syncthreads();
  constexpr int TPR = D / 4;  // threads per row, four numerators each
  const int d = 4 * (threadIdx.x % TPR);
  for (int r = threadIdx.x / TPR; r < x.rows; r += L::NT / TPR) {
    float mw[L::WAVES], mx = kNegInf, lt = 0.f;
#pragma unroll
    for (int w = 0; w < L::WAVES; ++w) {
      mw[w] = ml[(w * 32 + r) * 2];
      mx = fmaxf(mx, mw[w]);
    }
    f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < L::WAVES; ++w) {
      const float f = move_factor(mw[w], mx, c);
      lt += ml[(w * 32 + r) * 2 + 1] * f;
      // an empty wave's numerator is 0, and 0 times an empty factor stays 0
      y += *reinterpret_cast<const f32x4*>(num + (w * 32 + r) * L::OLD + d) * f;
    }
    const int tk = (int)a.group.div(x.r0 + r), hr = h * a.G + x.r0 + r - tk * a.G;
    const int64_t i = (int64_t)(x.row0 + tk) * a.Hq + hr;
    if (x.split) {
      const int64_t rows = a.N * a.Hq;
      if (d == 0) {
        a.part[2 * (i * a.splits + split)] = mx;
        a.part[2 * (i * a.splits + split) + 1] = lt;
      }
      *reinterpret_cast<f32x4*>(a.part + ((2 * rows * a.splits + 3) & ~(int64_t)3) + (i * a.splits + split) * D + d) = y;
    } else {
      uint16_t* orow = a.o + (int64_t)(x.row0 + tk) * a.o_t + (int64_t)hr * a.o_h;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = finish(y[e], lt, a.normalize);
      if (d < a.d) *reinterpret_cast<u32x2*>(orow + d) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      if (d == 0) row_stats(a, i, mx, lt);
    }
  }
}

template <int D, bool WIDE>
int32_t launch(const PagedArgs& a, int64_t tiles, hipStream_t s) {
  using L = Few<D, WIDE>;
  static bool done[kDevices] = {};
  const int32_t r = allow_lds(reinterpret_cast<const void*>(&paged_few_kernel<D, WIDE>), L::BYTES, done);
  if (r != CATOPT_OK) return r;
  const int64_t blocks = tiles * a.splits * a.Hkv;
  if (!grid_fits(blocks, L::NT)) return CATOPT_E_UNSUPPORTED;
  paged_few_kernel<D, WIDE><<<dim3((uint32_t)blocks), dim3(L::NT), L::BYTES, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_few_launch(const PagedArgs& a, int D, bool wide, int64_t tiles, hipStream_t s) {
  if (D == 128) return wide ? launch<128, true>(a, tiles, s) : launch<128, false>(a, tiles, s);
  return wide ? launch<64, true>(a, tiles, s) : launch<64, false>(a, tiles, s);
}

}  // namespace catopt
