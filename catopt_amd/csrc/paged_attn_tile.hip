// Paged attention with many query rows per key head (prompts and chunks): the
// tile loop of the contiguous 32-query kernel over cache pages.
//
// One workgroup = 4 waves = 128 rows of one key head, 32 per wave, a token's G
// query heads in neighbouring rows, so that they share every K and V tile.
// S^T = K Q^T and O^T += V^T P^T on the 32x32x16 MFMA: the accumulator's
// column is the query row, and the softmax statistics are lane-local.  Tiles
// of 64 keys are double buffered in LDS; each 1 KB of one comes by a direct
// global->LDS load whose 4 or 8 rows lie in one page, through a buffer
// resource of its own that ends behind the last key.
//
// A tile runs as two key halves of 32, each its own online-softmax step, so
// that the exponentials of one half issue between the MFMAs of the other.  The
// reference max moves only when a half exceeds it by kLazy (log2 units);
// until then p <= 2^kLazy, exact in range for fp32 and bf16.  The row's sum takes p
// in fp32; the product with V takes it rounded to bf16, which MFMA at this rate
// asks for: each term is off by half a step at most, and the result by 0.0021 to
// 0.0023 of its size on random inputs where its own rounding alone gives 0.0017.
//
// MFMAs and softmax VALU bound it together (0.39 and 0.48 of the cycles): four
// prompts of 4096, 32 heads of 128, 621 us, 886 TFLOP/s at a clock of 1.9 GHz (598
// to 657 from one card to another); 2048 tokens over 8192 keys, 32 heads on 8, 263 us
// (257 to 287).  Two workgroups a CU at D = 128 (registers),
// three at 64 (two: 77 us where three take 70, four prompts of 2048, 16 heads;
// four spill).  Further stages of tiles in flight measured level.
//
// The grid takes the key heads of a tile next to each other: consecutive
// workgroups go to the 8 XCDs in turn, so with a multiple of 8 key heads each
// XCD's L2 serves its own heads.  Tiles go from the last one down, which
// starts the longest of a causal sequence first.
#include <type_traits>

#include "paged_attn.hpp"

namespace catopt {
namespace {

constexpr int NT = 256;  // 4 waves
constexpr int KVB = 64;  // keys per tile
constexpr float kLazy = 8.0f;

template <int D>
struct TileLds {
  static constexpr int TILE = KVB * AttnRow<D>::BYTES, STAGE = 2 * TILE, BYTES = 2 * STAGE;
  static constexpr int LOADS = TILE / 4096;  // 1 KB loads of K (and of V) per wave
  static constexpr int ROWS = 1024 / AttnRow<D>::BYTES;  // rows of one
};

// Masks, odd values and moves of the maximum leave the loop's straight line: 1500
// new tokens over 4500 keys, 32 heads on 8, 142 -> 134 us; prompts of 4 x 4096 612
// -> 597.  (A macro: the hint does not survive a function's inlining.)
#define UNLIKELY(x) __builtin_expect(!!(x), 0)

// An empty asm use: the value is computed before this point.
__device__ __forceinline__ void pin(const bf16x8& x) { asm volatile("" ::"v"(__builtin_bit_cast(u32x4, x))); }
__device__ __forceinline__ void pin(float x) { asm volatile("" ::"v"(x)); }

template <int D>
__global__ __launch_bounds__((NT), (D == 64 ? 3 : 2)) void paged_tile_kernel(PagedArgs a, int tiles) {
  using L = TileLds<D>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int h, tr, split;
  decode_block(a, h, tr, split);
  PagedTile x = paged_tile<kTileRows>(a, tiles - 1 - tr);
  if (x.rows == 0) return;
  paged_ranges(a, x);
  if (!has_range(x, split)) return;
  const float c = a.scale * kLog2e;

  const int row = x.r0 + 32 * wave + l32, tok = (int)a.group.div(row), hq = h * a.G + row - tok * a.G;
  const bool live = 32 * wave + l32 < x.rows;
  const int lim = min(x.off + tok, x.len - 1);  // last key this row sees
  // of the wave's rows the first sees the fewest keys, the last the most
  const int w0 = x.r0 + 32 * wave, w1 = min(w0 + 31, x.r0 + x.rows - 1);
  const int lim0 = __builtin_amdgcn_readfirstlane(x.off + (int)a.group.div(w0));
  const int lim1 = __builtin_amdgcn_readfirstlane(x.off + (int)a.group.div(max(w1, 0)));
  const bool wave_live = 32 * wave < x.rows;

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m_run = kNegInf, m_true = kNegInf, l_run = 0.f;  // maxima in units of q . k

  const int k_end = min(x.kend, (split + 1) * x.keys);
  const int t0 = split * x.keys / KVB, t1 = (k_end + KVB - 1) / KVB;
  const int wave_end = wave_live ? min(k_end, lim1 + 1) : 0;
  const int32_t* table = a.table + (int64_t)x.b * a.table_ld;
  const uint16_t *kb = a.k + (int64_t)h * a.k_h, *vb = a.v + (int64_t)h * a.v_h;
  // a lane's 16 bytes of load i: tile row (4 i + wave) ROWS + sub, whose place
  // in its 8 keys and whose swizzles do not depend on i
  const int sub = lane / AttnRow<D>::CH, cp = lane % AttnRow<D>::CH, trow = wave * L::ROWS + sub;
  const uint32_t koff = group_offset(a.k_s, trow & 7, cp ^ (trow & (AttnRow<D>::CH - 1) & 15), a.d);
  const uint32_t voff = group_offset(a.v_s, trow & 7, cp ^ vswz<D>(trow), a.d);
  const uint32_t lds0 = lds_u32(lds) + wave * 1024;
  // the lanes hold the places of eight tiles, lane 8 i + j keys 8 j on of the
  // i-th; the page ids of the next eight are loaded one tile before they are used
  KeyGroup at{};
  uint64_t bads = 0;
  int next_page = -1;
  auto key_of = [&](int t) { return t * KVB + 8 * lane; };  // of the eight tiles from t on
  auto places = [&](int t) {
    bool odd;
    at = key_group(a, kb, vb, next_page, key_of(t), x.len, odd);
    bads = __ballot(odd);
  };
  auto issue = [&](int t, int stage) {
    const int lane0 = 8 * ((t - t0) & 7);
#pragma unroll
    for (int i = 0; i < L::LOADS; i += 2) {
      const int l0 = lane0 + ((4 * i + wave) * L::ROWS >> 3), l1 = lane0 + ((4 * i + 4 + wave) * L::ROWS >> 3);
      const uint32_t to = lds0 + stage * L::STAGE + i * 4096;
      dma_rows4(k_rsrc(at, l0), k_rsrc(at, l1), koff, to, v_rsrc(at, l0), v_rsrc(at, l1), voff, to + L::TILE, 4096);
    }
  };

  uint32_t bad = 0, bad_next = 0;  // a bit for each 8 keys of the tile whose page is invalid
  bf16x8 qf[D / 16];
  if (t0 < t1) {
    // the first pages' ids, the queries and the first tile are on their way
    // together; the queries as whole rows through the second stage, four times
    // fewer lines a load than as fragments
    next_page = group_page(a, table, key_of(t0), x.len);
    const uint64_t q = reinterpret_cast<uint64_t>(a.q + (int64_t)(x.row0 + tok) * a.q_t + (int64_t)hq * a.q_h);
    u32x4 qr[2 * L::LOADS];
#pragma unroll
    for (int i = 0; i < 2 * L::LOADS; ++i) {
      const int r = i * L::ROWS + sub;
      const uint32_t lo = __shfl((uint32_t)q, r, 64), hi = __shfl((uint32_t)(q >> 32), r, 64);
      qr[i] = u32x4{0, 0, 0, 0};
      if (32 * wave + r < x.rows && 8 * cp < a.d)
        qr[i] = *reinterpret_cast<const u32x4*>((((uint64_t)hi << 32) | lo) + 16 * cp);
    }
    places(t0);
    bad = (uint32_t)bads & 0xffu;
    issue(t0, 0);
    char* Qs = lds + L::STAGE + wave * 32 * AttnRow<D>::BYTES;
#pragma unroll
    for (int i = 0; i < 2 * L::LOADS; ++i) *reinterpret_cast<u32x4*>(Qs + tile_off<D>(i * L::ROWS + sub, cp)) = qr[i];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) qf[j] = *reinterpret_cast<const bf16x8*>(Qs + tile_off<D>(l32, 2 * j + g));
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }

  auto tile = [&](int t, auto stage_tag) {
    constexpr int cur = decltype(stage_tag)::value;
    if (t + 1 < t1) {
      const int in = (t + 1 - t0) & 7;
      if (in == 0) places(t + 1);
      bad_next = (uint32_t)(bads >> (8 * in)) & 0xffu;
      issue(t + 1, cur ^ 1);
      if (in == 6) next_page = group_page(a, table, key_of(t + 3), x.len);
    }
    const char* Ks = lds + cur * L::STAGE;
    const char* Vs = Ks + L::TILE;
    const int kv0 = t * KVB;
    if (kv0 < wave_end) {
      //   QK(0) | max(0) | QK(1) + exp(0) | max(1) | PV(0) + exp(1) | PV(1)
      const bool masked = kv0 + KVB > x.len || kv0 + KVB - 1 > lim0 || bad;
      bf16x8 kf[2][D / 16], vf[2][D / 16];
      auto read_k = [&](int kb2) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          kf[kb2][j] = *reinterpret_cast<const bf16x8*>(Ks + tile_off<D>(32 * kb2 + l32, 2 * j + g));
      };
      auto qk = [&](int kb2, f32x16& s) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) s = mfma32x32x16(kf[kb2][j], qf[j], s);
      };
      auto pv = [&](int kb2, const bf16x8* p) {
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
          for (int u = 0; u < 2; ++u) acc[db] = mfma32x32x16(vf[kb2][2 * db + u], p[u], acc[db]);
      };
      auto apply_mask = [&](int kb2, f32x16& s) { mask_scores(s, lim - kv0 - 32 * kb2, (bad >> (4 * kb2)) & 15u); };
      // row max of a half over both lane halves, the true max, and the lazy
      // move of the reference max; returns the factor for O^T (1: no move)
      auto half_max = [&](const f32x16& s) -> float {
        float mt = kNegInf;
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[r]);
        {
          const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mt),
                                                           __builtin_bit_cast(uint32_t, mt), false, false);
          mt = fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]));
        }
        m_true = fmaxf(m_true, mt);
        float alpha = 1.f;
        if (UNLIKELY(__builtin_amdgcn_ballot_w64((mt - m_run) * c > kLazy) != 0)) {
          const float m_new = fmaxf(m_run, mt);
          alpha = move_factor(m_run, m_new, c);
          l_run *= alpha;
          m_run = m_new;
        }
        return alpha;
      };
      auto rescale = [&](float alpha) {
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
      };
      auto half_exp = [&](const f32x16& s, bf16x8* p) {
        const float mc = (m_run == kNegInf ? 0.f : m_run) * c;
        float lsum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -mc));
          lsum += e;
          p[r >> 3][r & 7] = static_cast<__bf16>(e);
        }
        l_run += lsum;
      };

      f32x16 s0, s1;
      bf16x8 p0[2], p1[2];
      read_k(0);
      read_k(1);
      qk(0, s0);
      if (UNLIKELY(masked)) apply_mask(0, s0);
      const float a0 = half_max(s0);
      if (UNLIKELY(__builtin_amdgcn_ballot_w64(a0 != 1.f) != 0)) rescale(a0);
      __builtin_amdgcn_sched_barrier(0);
      qk(1, s1);
      half_exp(s0, p0);
      read_v<D>(Vs, 0, vf[0]);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // VALU
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // DS read
      }
      pin(p0[0]);
      pin(p0[1]);
      pin(l_run);
      __builtin_amdgcn_sched_barrier(0);
      if (UNLIKELY(masked)) apply_mask(1, s1);
      const float a1 = half_max(s1);
      if (UNLIKELY(masked) && UNLIKELY(odd_values<D>(vf[0]))) take_odd_values<D>(vf[0], lim - kv0, bad & 15u, acc);
      __builtin_amdgcn_sched_barrier(0);
      pv(0, p0);
      half_exp(s1, p1);
      read_v<D>(Vs, 32, vf[1]);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // VALU
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // DS read
      }
      pin(p1[0]);
      pin(p1[1]);
      pin(l_run);
      __builtin_amdgcn_sched_barrier(0);
      if (UNLIKELY(__builtin_amdgcn_ballot_w64(a1 != 1.f) != 0)) rescale(a1);
      if (UNLIKELY(masked) && UNLIKELY(odd_values<D>(vf[1]))) take_odd_values<D>(vf[1], lim - kv0 - 32, (bad >> 4) & 15u, acc);
      pv(1, p1);
    }
    bad = bad_next;
    if (t + 1 < t1) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
  };
  for (int t = t0; t < t1; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>{});
  }

  // ---- epilogue: back to the true max, then the row or its range's carrier
  const float fix = m_true != kNegInf && m_run != kNegInf ? __builtin_amdgcn_exp2f((m_run - m_true) * c) : 1.f;
  const float l_sum = l_run + __shfl_xor(l_run, 32, 64);
  const int64_t i = (int64_t)(x.row0 + tok) * a.Hq + hq;
  if (x.split) {
    if (!live) return;
    const int64_t rows = a.N * a.Hq, at = i * a.splits + split;
    if (g == 0) {
      a.part[2 * at] = m_true;
      a.part[2 * at + 1] = l_sum * fix;
    }
    float* num = a.part + ((2 * rows * a.splits + 3) & ~(int64_t)3) + at * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg)
        *reinterpret_cast<f32x4*>(num + 32 * db + 8 * rg + 4 * g) =
            f32x4{acc[db][4 * rg] * fix, acc[db][4 * rg + 1] * fix, acc[db][4 * rg + 2] * fix, acc[db][4 * rg + 3] * fix};
    return;
  }
  // the lane halves swap words, so that each stores 16 bytes: 8 columns of an
  // even (g = 0) or odd eighth of every 32
  uint16_t* orow = a.o + (int64_t)(x.row0 + tok) * a.o_t + (int64_t)hq * a.o_h;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
#pragma unroll
    for (int rg = 0; rg < 4; rg += 2) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x16& y = acc[db];
        const int r = 4 * rg + 2 * e;
        const auto sw = __builtin_amdgcn_permlane32_swap(
            pack_bf16x2(finish(y[r], l_sum, a.normalize), finish(y[r + 1], l_sum, a.normalize)),
            pack_bf16x2(finish(y[r + 4], l_sum, a.normalize), finish(y[r + 5], l_sum, a.normalize)), false, false);
        w[e] = sw[0], w[2 + e] = sw[1];
      }
      const int d = 32 * db + 8 * (rg + g);
      if (live && d < a.d) *reinterpret_cast<u32x4*>(orow + d) = w;
    }
  }
  if (live && g == 0) row_stats(a, i, m_true, l_sum * fix);
}

template <int D>
int32_t launch(const PagedArgs& a, int64_t tiles, hipStream_t s) {
  static bool done[kDevices] = {};
  const int32_t r = allow_lds(reinterpret_cast<const void*>(&paged_tile_kernel<D>), TileLds<D>::BYTES, done);
  if (r != CATOPT_OK) return r;
  const int64_t blocks = tiles * a.splits * a.Hkv;
  if (!grid_fits(blocks, NT)) return CATOPT_E_UNSUPPORTED;
  paged_tile_kernel<D><<<dim3((uint32_t)blocks), dim3(NT), TileLds<D>::BYTES, s>>>(a, (int)tiles);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_tile_launch(const PagedArgs& a, int D, int64_t tiles, hipStream_t s) {
  return D == 128 ? launch<128>(a, tiles, s) : launch<64>(a, tiles, s);
}

}  // namespace catopt
