// Eviction from a paged cache by accumulated attention weight: per (sequence,
// key head) the last `recent` keys and the largest weights of the others stay,
// then the kept rows move to other pages.
#include "paged.hpp"

namespace catopt {
namespace {

struct EvictArgs {
  Pages k, v, ko, vo;
  const int32_t *table, *out_table, *lens;
  const float* w;
  float* w_out;
  int32_t *kept, *new_lens;
  int64_t table_ld, out_ld, w_b, w_h, wo_b, wo_h, n_pages, n_out_pages;
  FastDiv page, out_page;
  int B, H, cap, budget, recent, row16;  // row16: 16-byte pieces of a row
};

constexpr int NT = 1024;

// A total order of floats as unsigned: NaN above every number, -0 equal to 0.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kWaves = NT / 64, kRegs = 16;  // weights per lane held in registers: NT * kRegs keys
constexpr int kBins = 2048;

// One workgroup per (sequence, head); wave i takes the i-th of 16 runs of the
// keys.  A radix select by 11, 11 and 10 bits of the rank finds the rank of the
// last key that stays and how many of its equals do (the first ones); each wave
// then counts its keys above and at that rank, one exchange of the counts gives
// every wave its place, and a second sweep lists the kept keys in order.
// HELD: a lane's weights stay in registers over the five sweeps (they cover
// tables of up to 16384 keys); else each sweep reads them again, from L2.
template <bool HELD>
__global__ __launch_bounds__(NT) void evict_select(EvictArgs a) {
  __shared__ uint32_t hist[kBins], wave_sum[kWaves], sh_bin, sh_left, cnt_above[kWaves], cnt_equal[kWaves];
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = min(max(a.lens[b], 0), a.cap), m = min(n, a.budget);
  const int old = n - min(a.recent, m);  // keys from here on stay
  const float* w = a.w + b * a.w_b + h * a.w_h;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = m;
  const int steps = (n + NT - 1) / NT, first = wave * steps * 64;  // this wave's keys: `steps` of 64

  // weights of the U steps from step i0 on: the loads take a valid address
  // whatever the step, so that none waits for another
  auto load = [&](int i0, auto& x) {
    constexpr int U = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = n > 0 ? w[min(first + 64 * (i0 + i) + lane, n - 1)] : 0.f;
  };
  float held[HELD ? kRegs : 1];
  if (HELD) load(0, held);
  // f(key, rank, weight) for every key of the wave
  auto sweep = [&](auto f) {
    if (HELD) {
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (i < steps) f(first + 64 * i + lane, rank_of(held[i]), held[i]);
    } else {
      constexpr int U = 8;
      for (int i0 = 0; i0 < steps; i0 += U) {
        float x[U];
        load(i0, x);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (i0 + i < steps) f(first + 64 * (i0 + i) + lane, rank_of(x[i]), x[i]);
      }
    }
  };

  // of the first `old` keys `need` stay: those above the rank `limit` and the
  // first `equals` of that rank
  const uint32_t need = (uint32_t)(m - (n - old));
  uint32_t limit = 0, equals = need;
  const bool some = need > 0 && need < (uint32_t)old;
  if (some) {
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
      const uint32_t mask = round == 0 ? 0u : round == 1 ? 0xffe00000u : 0xfffffc00u;
      hist[tid] = 0;
      hist[tid + NT] = 0;
      __syncthreads();
      sweep([&](int j, uint32_t r, float) {
        if (j < old && (r & mask) == limit) atomicAdd(&hist[(r >> shift) & ((1u << bits) - 1)], 1u);
      });
      __syncthreads();
      // keys in this thread's two bins and in all bins above them
      const uint32_t hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
      uint32_t sum = hi + lo;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
      }
      if (lane == 63) wave_sum[wave] = sum;
      __syncthreads();
      uint32_t above = sum - hi - lo;
      for (int i = 0; i < wave; ++i) above += wave_sum[i];
      if (above < equals && equals <= above + hi + lo) {  // one thread
        const bool in_hi = equals <= above + hi;
        sh_bin = kBins - 1 - 2 * tid - (in_hi ? 0 : 1);
        sh_left = equals - above - (in_hi ? 0u : hi);
      }
      __syncthreads();
      limit |= sh_bin << shift;
      equals = sh_left;
    }
  } else if (need == 0) {
    limit = 0xffffffffu, equals = 0;  // none of them stays
  }  // else all do: every rank is at least 0, and all `need` of rank 0 would stay

  uint32_t na = 0, ne = 0;
  sweep([&](int j, uint32_t r, float) {
    const bool is_old = j < old;
    na += __popcll(__ballot(j < n && (!is_old || r > limit)));
    ne += __popcll(__ballot(is_old && r == limit));
  });
  if (lane == 0) cnt_above[wave] = na, cnt_equal[wave] = ne;
  __syncthreads();
  uint32_t at = 0, eq = 0;  // kept keys, and keys at the limit, before this wave's
  for (int i = 0; i < wave; ++i) {
    at += cnt_above[i] + (eq < equals ? min(cnt_equal[i], equals - eq) : 0u);
    eq += cnt_equal[i];
  }
  const uint64_t below = (1ull << lane) - 1;
  float* w_out = a.w_out ? a.w_out + b * a.wo_b + h * a.wo_h : nullptr;
  sweep([&](int j, uint32_t r, float x) {
    const bool is_old = j < old;
    const uint64_t be = __ballot(is_old && r == limit);
    const bool stay = j < n && (!is_old || r > limit || (r == limit && eq + __popcll(be & below) < equals));
    const uint64_t bs = __ballot(stay);
    const uint32_t to = at + __popcll(bs & below);
    if (stay && to < (uint32_t)m) {
      kept[to] = j;
      if (HELD && w_out) w_out[to] = x;  // every wave holds its own: they may lie where the weights did
    }
    at += __popcll(bs);
    eq += __popcll(be);
  });
  for (int j = m + tid; j < a.budget; j += NT) kept[j] = -1;
  if (HELD || !w_out) return;
  // the kept weights, which may go where the weights are: a kept key's place is
  // never behind it, so a step's writes lie before every later step's reads
  __syncthreads();
  for (int i0 = 0; i0 < m; i0 += NT) {
    const int i = i0 + tid;
    const float x = i < m ? w[kept[i]] : 0.f;
    __syncthreads();
    if (i < m) w_out[i] = x;
  }
}

// 16 bytes of one kept row of k and of v per thread.  They are read for the last
// time, so the loads leave the caches alone (8 x 8 heads, 2048 keys each: 48 -> 43 us
// for the whole call).
__global__ __launch_bounds__(256) void evict_move(EvictArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / a.row16;
  const int piece = (int)(at - row * a.row16);
  if (row >= (int64_t)a.B * a.H * a.budget) return;
  const int64_t bh = row / a.budget;
  const int i = (int)(row - bh * a.budget), b = (int)(bh / a.H), h = (int)(bh - (int64_t)b * a.H);
  const int j = a.kept[row];
  if (j < 0) return;
  const uint32_t tp = a.out_page.div(i), sp = a.page.div(j);
  const int64_t to = a.out_table[b * a.out_ld + tp], from = a.table[b * a.table_ld + sp];
  if (to < 0 || to >= a.n_out_pages) return;
  const uint32_t ti = i - tp * a.out_page.d, si = j - sp * a.page.d;
  u32x4 k = u32x4{0, 0, 0, 0}, v = u32x4{0, 0, 0, 0};
  if (from >= 0 && from < a.n_pages) {  // strides in 16-byte pieces
    k = __builtin_nontemporal_load(static_cast<const u32x4*>(a.k.p) + (from * a.k.s_page + h * a.k.s_head + si * a.k.s_slot + piece));
    v = __builtin_nontemporal_load(static_cast<const u32x4*>(a.v.p) + (from * a.v.s_page + h * a.v.s_head + si * a.v.s_slot + piece));
  }
  static_cast<u32x4*>(const_cast<void*>(a.ko.p))[to * a.ko.s_page + h * a.ko.s_head + ti * a.ko.s_slot + piece] = k;
  static_cast<u32x4*>(const_cast<void*>(a.vo.p))[to * a.vo.s_page + h * a.vo.s_head + ti * a.vo.s_slot + piece] = v;
}

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int32_t catopt_hip_paged_evict(int32_t dtype, int64_t B, int64_t Hkv, int64_t d, const void* k_pages,
                                          const void* v_pages, int64_t n_pages, int64_t page_size,
                                          const int32_t* block_table, int64_t table_ld, int64_t n_table,
                                          const int32_t* kv_lens, const float* weights, int64_t budget, int64_t recent,
                                          void* k_out, void* v_out, int64_t n_out_pages, int64_t out_page_size,
                                          const int32_t* out_table, int64_t out_table_ld, int64_t n_out_table,
                                          int32_t* kept, int32_t* new_lens, float* weights_out,
                                          const int64_t* strides, void* stream) {
  if (dtype != CATOPT_F32 && dtype != CATOPT_BF16) return CATOPT_E_UNSUPPORTED;
  if (B < 0 || Hkv < 1 || d < 1 || n_pages < 0 || page_size < 1 || n_table < 0 || table_ld < 0)
    return CATOPT_E_INVAL;
  if (n_out_pages < 0 || out_page_size < 1 || n_out_table < 0 || out_table_ld < 0) return CATOPT_E_INVAL;
  if (budget < 1 || recent < 0 || recent > budget) return CATOPT_E_INVAL;
  const int64_t row = d * (dtype == CATOPT_BF16 ? 2 : 4), lim = 1LL << 30;
  if (row % 16 || row > (1 << 14)) return CATOPT_E_UNSUPPORTED;
  if (page_size > lim || out_page_size > lim || n_table > lim || n_out_table > lim || budget > lim || B > (1 << 20) || Hkv > (1 << 20))
    return CATOPT_E_UNSUPPORTED;
  if (n_table * page_size > lim || !grid_fits(B * Hkv, NT)) return CATOPT_E_UNSUPPORTED;  // B Hkv < 2^22
  if (n_out_table * out_page_size < budget) return CATOPT_E_INVAL;
  if (B == 0) return CATOPT_OK;
  const int64_t step = 16 / (dtype == CATOPT_BF16 ? 2 : 4);
  if (!strides || !strides_fit(strides, 12, step) || !strides_fit(strides + 12, 4, 1)) return CATOPT_E_INVAL;
  if (!kv_lens || !kept || !new_lens || !out_table || (n_table > 0 && (!block_table || !weights))) return CATOPT_E_INVAL;
  if ((n_pages > 0 && (!k_pages || !v_pages)) || (n_out_pages > 0 && (!k_out || !v_out))) return CATOPT_E_INVAL;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out)) return CATOPT_E_INVAL;
  const int64_t* s = strides;
  const int64_t size = 16 / step;
  const Layout lk = layout_pages(k_pages, size, n_pages, Hkv, page_size, d, s);
  const Layout lv = layout_pages(v_pages, size, n_pages, Hkv, page_size, d, s + 3);
  const Layout ko = layout_pages(k_out, size, n_out_pages, Hkv, out_page_size, d, s + 6);
  const Layout vo = layout_pages(v_out, size, n_out_pages, Hkv, out_page_size, d, s + 9);
  const Layout w = layout3(weights, 4, B, s[12], Hkv, s[13], n_table * page_size);
  const Layout wo = layout3(weights_out, 4, B, s[14], Hkv, s[15], budget);
  // the same pool keeps its place in both roles; keys and values may be parts
  // of one storage, so only their beginnings tell them apart
  const bool pool = k_out == k_pages;
  if (ko.folded() || vo.folded() || (!ko.empty() && (k_out == v_out || k_out == v_pages || v_out == k_pages)))
    return CATOPT_E_INVAL;
  if (pool ? !ko.same(lk) || !vo.same(lv) || n_out_pages != n_pages || (n_table > 0 && out_table == block_table)
           : ko.overlaps(lk) || vo.overlaps(lv))
    return CATOPT_E_INVAL;
  if (ko.overlaps(w) || vo.overlaps(w) || ko.overlaps(wo) || vo.overlaps(wo) || lk.overlaps(wo) || lv.overlaps(wo))
    return CATOPT_E_INVAL;
  if (wo.folded() || (wo.overlaps(w) && !wo.same(w))) return CATOPT_E_INVAL;
  EvictArgs a{};
  a.k = Pages{k_pages, s[0] / step, s[1] / step, s[2] / step};
  a.v = Pages{v_pages, s[3] / step, s[4] / step, s[5] / step};
  a.ko = Pages{k_out, s[6] / step, s[7] / step, s[8] / step};
  a.vo = Pages{v_out, s[9] / step, s[10] / step, s[11] / step};
  a.w = weights, a.w_out = weights_out, a.kept = kept, a.new_lens = new_lens;
  a.w_b = s[12], a.w_h = s[13], a.wo_b = s[14], a.wo_h = s[15];
  a.table = block_table, a.out_table = out_table, a.lens = kv_lens, a.table_ld = table_ld, a.out_ld = out_table_ld;
  a.n_pages = n_pages, a.n_out_pages = n_out_pages;
  a.page = FastDiv::of(page_size), a.out_page = FastDiv::of(out_page_size);
  a.B = (int)B, a.H = (int)Hkv, a.cap = (int)(n_table * page_size), a.budget = (int)budget, a.recent = (int)recent;
  a.row16 = (int)(row / 16);
  const int64_t blocks = (B * Hkv * budget * a.row16 + 255) / 256;  // the product is below 2^62
  if (!grid_fits(blocks, 256)) return CATOPT_E_UNSUPPORTED;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.cap <= NT * kRegs)
    evict_select<true><<<dim3((uint32_t)(B * Hkv)), dim3(NT), 0, st>>>(a);
  else
    evict_select<false><<<dim3((uint32_t)(B * Hkv)), dim3(NT), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  evict_move<<<dim3((uint32_t)blocks), dim3(256), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}
