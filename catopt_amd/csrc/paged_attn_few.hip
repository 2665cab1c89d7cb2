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
// V go global->LDS directly, one stage ahead; a 1 KB load covers 4 or 8 rows,
// which lie in one page, so each has a buffer resource of its own whose range
// ends behind the last key.  The page ids of a stage are loaded one stage
// before its rows.
#include "paged_attn.hpp"

namespace catopt {
namespace {

template <int D>
struct Few {
  static constexpr int WAVES = D == 128 ? 2 : 4, NT = 64 * WAVES;
  static constexpr int KEYS = 32 * WAVES;              // per stage
  static constexpr int HALF = 32 * AttnRow<D>::BYTES;  // a wave's K (or V) rows of a stage
  static constexpr int WAVE_BYTES = 2 * HALF, STAGE = WAVES * WAVE_BYTES, BYTES = 2 * STAGE;
  static constexpr int LOADS = HALF / 1024;            // 1 KB loads of K (and of V) per stage
  static constexpr int ROWS = 32 / LOADS;              // rows of one
  static constexpr int OLD = D + 4;                    // row of the merge buffer, floats
  static_assert(WAVES * 32 * OLD * 4 + WAVES * 64 * 4 <= BYTES, "the merge reuses the stages");
};

template <int D>
__global__ __launch_bounds__(Few<D>::NT, 2) void paged_few_kernel(PagedArgs a) {
  using L = Few<D>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.Hkv, ts = blockIdx.x / a.Hkv, t = ts / a.splits, split = ts - t * a.splits;
  PagedTile x = paged_tile<kFewRows>(a, t);
  if (x.rows == 0) return;
  paged_ranges(a, x);
  if (split >= x.splits) return;
  const float c = a.scale * kLog2e;

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
  const int lim = x.off + tok;  // last key this row sees

  const int k_end = min(x.kend, (split + 1) * x.keys);
  const int t0 = split * x.keys / L::KEYS, t1 = (k_end + L::KEYS - 1) / L::KEYS;
  const int32_t* table = a.table + (int64_t)x.b * a.table_ld;
  const uint16_t *kb = a.k + (int64_t)h * a.k_h, *vb = a.v + (int64_t)h * a.v_h;
  // a lane's 16 bytes of a load: row lane / CH of it.  The swizzles depend on a
  // row's place among 16 (K, D = 128: loads i and i + 4 agree), 8 or 4 rows.
  // Columns past d lie outside every resource.
  const int sub = lane / AttnRow<D>::CH, cp = lane % AttnRow<D>::CH;
  uint32_t koff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kc = cp ^ ((i * L::ROWS + sub) & (AttnRow<D>::CH - 1) & 15);
    koff[i] = kc * 8 < a.d ? (uint32_t)(sub * (int)a.k_s + kc * 8) * 2u : 0x7ffffff0u;
  }
  const int vc = cp ^ vswz<D>(sub);
  const uint32_t voff = vc * 8 < a.d ? (uint32_t)(sub * (int)a.v_s + vc * 8) * 2u : 0x7ffffff0u;
  const uint32_t lds0 = lds_u32(lds) + wave * L::WAVE_BYTES;
  auto issue = [&](int st, int stage, const PageIds& ids) {
    const int key0 = st * L::KEYS + 32 * wave;
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
      const int grp = i * L::ROWS / 8;
      const int page = __builtin_amdgcn_readlane(ids.page, grp);
      const int slot = __builtin_amdgcn_readlane(ids.slot, grp) + i * L::ROWS % 8;
      const int rows = min(x.len - (key0 + i * L::ROWS), L::ROWS);
      dma_buf(page_rsrc(kb, page, slot, a.k_p, a.k_s, rows, a.d, a.n_pages), koff[i & 3], lds0 + stage * L::STAGE + i * 1024);
      dma_buf(page_rsrc(vb, page, slot, a.v_p, a.v_s, rows, a.d, a.n_pages), voff,
              lds0 + stage * L::STAGE + L::HALF + i * 1024);
    }
  };

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m = kNegInf, l = 0.f;
  float* srow = a.scores ? a.scores + ((int64_t)(x.row0 + tok) * a.Hq + hq) * a.cap : nullptr;

  PageIds ids{-1, 0}, next{-1, 0};
  uint32_t bad = 0, bad_next = 0;
  if (t0 < t1) {
    ids = page_ids(a, table, t0 * L::KEYS + 32 * wave, x.len);
    bad = bad_groups(a, ids, t0 * L::KEYS + 32 * wave, x.len) & 15u;
    issue(t0, 0, ids);
    next = page_ids(a, table, (t0 + 1) * L::KEYS + 32 * wave, x.len);
  }
  for (int st = t0; st < t1; ++st) {
    const int stage = (st - t0) & 1;
    // this stage has landed (for every wave: an LDS-DMA write is read only past
    // a barrier), and every wave is done with the other half of the ring
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (st + 1 < t1) {
      bad_next = bad_groups(a, next, (st + 1) * L::KEYS + 32 * wave, x.len) & 15u;
      issue(st + 1, stage ^ 1, next);
      next = page_ids(a, table, (st + 2) * L::KEYS + 32 * wave, x.len);
    }
    const int key0 = st * L::KEYS + 32 * wave;
    const uint32_t bad_now = bad;
    bad = bad_next;
    if (key0 >= k_end) continue;
    const char* Ks = lds + stage * L::STAGE + wave * L::WAVE_BYTES;
    const char* Vs = Ks + L::HALF;

    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      s = mfma32x32x16(*reinterpret_cast<const bf16x8*>(Ks + tile_off<D>(l32, 2 * j + g)), qf[j], s);
    // some row does not see some key: the first row sees the fewest
    const bool masked = key0 + 32 > x.len || key0 + 31 > x.off + x.r0 / a.G || bad_now;
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = key0 + acc_row(r, g);
        const bool keep = key < x.len && key <= lim && !((bad_now >> (acc_row(r, g) >> 3)) & 1);
        s[r] = keep ? s[r] : kNegInf;
      }
    }
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
    if (masked && odd_values<D>(vf)) take_odd_values<D>(vf, p, acc);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[db] = mfma32x32x16(vf[2 * db + u], p[u], acc[db]);
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
    if (x.splits > 1) {
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
      if (d == 0) {
        if (a.m_out) a.m_out[i] = mx * a.scale;
        if (a.l_out) a.l_out[i] = lt;
      }
    }
  }
}

template <int D>
int32_t launch(const PagedArgs& a, int64_t tiles, hipStream_t s) {
  static bool attr_done = false;  // idempotent; benign race (same value written)
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_few_kernel<D>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, Few<D>::BYTES);
    if (e != hipSuccess) return set_hip_error(e);
    attr_done = true;
  }
  const int64_t blocks = tiles * a.splits * a.Hkv;
  if (!grid_fits(blocks, Few<D>::NT)) return CATOPT_E_UNSUPPORTED;
  paged_few_kernel<D><<<dim3((uint32_t)blocks), dim3(Few<D>::NT), Few<D>::BYTES, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_few_launch(const PagedArgs& a, int D, int64_t tiles, hipStream_t s) {
  return D == 128 ? launch<128>(a, tiles, s) : launch<64>(a, tiles, s);
}

}  // namespace catopt
