// Eviction from a paged cache by accumulated attention weight: per (sequence,
// key head) the last `recent` keys and the largest weights of the others stay,
// and the kept rows move to other pages.
//
// One launch: `parts` workgroups per (sequence, head) each make the whole
// choice, which takes 10 us at 2048 keys and 16 at 16000, and move their share
// of the rows.  That takes 12 us for 2048 keys of one sequence, 8 heads, and 40
// for eight sequences of up to 16000 that keep 2048 (132 MB, so the move runs at
// 5.5 TB/s); a launch for the choice and one for the move take 2.6 and 1.4 more.
// HBM bounds the move, rounds of LDS atomics and barriers the choice.
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
  FastDiv row16;                      // 16-byte pieces of a row
  int B, H, cap, budget, recent, parts, clear;
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

// 16 bytes of each of U pieces of kept rows (of k and of v) per thread.  They
// are read for the last time, so the loads leave the caches alone.  (Two pieces:
// 40.5 us in the case above, 42.0 with four, 44.0 with eight.)
template <int U>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const int32_t* kept, int b, int h, int lo, int hi) {
  const int32_t *table = a.table + b * a.table_ld, *out_table = a.out_table + b * a.out_ld;
  const uint32_t pieces = (uint32_t)(hi - lo) * a.row16.d;
  for (uint32_t at0 = threadIdx.x; at0 < pieces; at0 += U * NT) {
    u32x4 k[U], v[U];
    int64_t to_k[U], to_v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = at0 + u * NT, r = a.row16.div(min(at, pieces - 1)), piece = min(at, pieces - 1) - r * a.row16.d;
      const int i = lo + (int)r, j = kept[i];
      const uint32_t tp = a.out_page.div(i), sp = a.page.div(j);
      const int64_t to = out_table[tp], from = table[sp];
      const int64_t ti = i - (int)(tp * a.out_page.d), si = j - (int)(sp * a.page.d);
      k[u] = v[u] = u32x4{0, 0, 0, 0};
      if (from >= 0 && from < a.n_pages) {  // strides in 16-byte pieces
        k[u] = __builtin_nontemporal_load(static_cast<const u32x4*>(a.k.p) +
                                          (from * a.k.s_page + h * a.k.s_head + si * a.k.s_slot + piece));
        v[u] = __builtin_nontemporal_load(static_cast<const u32x4*>(a.v.p) +
                                          (from * a.v.s_page + h * a.v.s_head + si * a.v.s_slot + piece));
      }
      const bool ok = at < pieces && to >= 0 && to < a.n_out_pages;
      to_k[u] = ok ? to * a.ko.s_page + h * a.ko.s_head + ti * a.ko.s_slot + piece : -1;
      to_v[u] = to * a.vo.s_page + h * a.vo.s_head + ti * a.vo.s_slot + piece;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (to_k[u] < 0) continue;
      static_cast<u32x4*>(const_cast<void*>(a.ko.p))[to_k[u]] = k[u];
      static_cast<u32x4*>(const_cast<void*>(a.vo.p))[to_v[u]] = v[u];
    }
  }
}

// Wave i of a workgroup takes the i-th of 16 runs of the keys.  A radix select by 11, 11 and 10 bits of the rank finds the rank of the
// last key that stays and how many of its equals do (the first ones); each wave
// then counts its keys above and at that rank, one exchange of the counts gives
// every wave its place, and a second sweep lists the kept keys in order.
// HELD: a lane's weights stay in registers over the five sweeps (they cover
// tables of up to 16384 keys); else each sweep reads them again, from L2.
template <bool HELD>
__global__ __launch_bounds__(NT) void evict_kernel(EvictArgs a) {
  __shared__ uint32_t hist[kBins], wave_sum[kWaves], sh_bin, sh_left, sh_all, cnt_above[kWaves], cnt_equal[kWaves];
  const int bh = blockIdx.x / a.parts, part = blockIdx.x - bh * a.parts;
  const int b = bh / a.H, h = bh - b * a.H, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = min(max(a.lens[b], 0), a.cap), m = min(n, a.budget);
  const int old = n - min(a.recent, m);  // keys from here on stay
  const float* w = a.w + b * a.w_b + h * a.w_h;
  int32_t* kept = a.kept + (int64_t)bh * a.budget;
  if (h == 0 && part == 0 && tid == 0) a.new_lens[b] = m;
  // this workgroup's kept keys
  const int share = (m + a.parts - 1) / a.parts, lo = min(part * share, m), hi = min(lo + share, m);
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
      const uint32_t upper = hist[kBins - 1 - 2 * tid], lower = hist[kBins - 2 - 2 * tid];
      uint32_t sum = upper + lower;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
      }
      if (lane == 63) wave_sum[wave] = sum;
      __syncthreads();
      uint32_t above = sum - upper - lower;
      for (int i = 0; i < wave; ++i) above += wave_sum[i];
      if (above < equals && equals <= above + upper + lower) {  // one thread
        const bool in_upper = equals <= above + upper;
        sh_bin = kBins - 1 - 2 * tid - (in_upper ? 0 : 1);
        sh_left = equals - above - (in_upper ? 0u : upper);
        sh_all = sh_left == (in_upper ? upper : lower);
      }
      __syncthreads();
      limit |= sh_bin << shift;
      equals = sh_left;
      if (sh_all) {  // the whole bin stays: all ranks from its first on, which is not 0 as need < old
        limit -= 1, equals = 0;
        break;
      }
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
    if (stay && to >= (uint32_t)lo && to < (uint32_t)hi) {
      kept[to] = j;
      // (one part alone may write where the weights are: its waves hold theirs)
      if (HELD && w_out) w_out[to] = x;
    }
    at += __popcll(bs);
    eq += __popcll(be);
  });
  if (part == 0)
    for (int j = m + tid; j < a.budget; j += NT) {
      kept[j] = -1;
      if (w_out && a.clear) w_out[j] = 0.f;
    }
  __syncthreads();  // the list is written
  if (!HELD && w_out) {
    // the kept weights, which one part alone may write where the weights are: a
    // kept key's place is never behind it, so a step's writes lie before every
    // later step's reads
    for (int i0 = lo; i0 < hi; i0 += NT) {
      const int i = i0 + tid;
      const float x = i < hi ? w[kept[i]] : 0.f;
      __syncthreads();
      if (i < hi) w_out[i] = x;
    }
  }
  move_rows<2>(a, kept, b, h, lo, hi);
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
                                          int32_t clear_behind, const int64_t* strides, void* stream) {
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
  // a head's kept rows are counted in 16-byte pieces, in 31 bits
  if ((budget < n_table * page_size ? budget : n_table * page_size) * (row / 16) > lim) return CATOPT_E_UNSUPPORTED;
  if (B == 0) return CATOPT_OK;
  const int64_t step = 16 / (dtype == CATOPT_BF16 ? 2 : 4);
  if (!strides) return CATOPT_E_INVAL;
  const Strides rows(strides, {n_pages, Hkv, page_size, n_pages, Hkv, page_size, n_out_pages, Hkv, out_page_size,
                               n_out_pages, Hkv, out_page_size}, step);
  const Strides sums(strides + 12, {B, Hkv, B, Hkv}, 1);
  if (!rows.fit || !sums.fit) return CATOPT_E_INVAL;
  if (!kv_lens || !kept || !new_lens || !out_table || (n_table > 0 && (!block_table || !weights))) return CATOPT_E_INVAL;
  if ((n_pages > 0 && (!k_pages || !v_pages)) || (n_out_pages > 0 && (!k_out || !v_out))) return CATOPT_E_INVAL;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out)) return CATOPT_E_INVAL;
  const int64_t *s = rows.s, *sw = sums.s;
  const int64_t size = 16 / step;
  const Layout lk = layout_pages(k_pages, size, n_pages, Hkv, page_size, d, s);
  const Layout lv = layout_pages(v_pages, size, n_pages, Hkv, page_size, d, s + 3);
  const Layout ko = layout_pages(k_out, size, n_out_pages, Hkv, out_page_size, d, s + 6);
  const Layout vo = layout_pages(v_out, size, n_out_pages, Hkv, out_page_size, d, s + 9);
  const Layout w = layout3(weights, 4, B, sw[0], Hkv, sw[1], n_table * page_size);
  const Layout wo = layout3(weights_out, 4, B, sw[2], Hkv, sw[3], budget);
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
  a.w_b = sw[0], a.w_h = sw[1], a.wo_b = sw[2], a.wo_h = sw[3];
  a.table = block_table, a.out_table = out_table, a.lens = kv_lens, a.table_ld = table_ld, a.out_ld = out_table_ld;
  a.n_pages = n_pages, a.n_out_pages = n_out_pages;
  a.page = FastDiv::of(page_size), a.out_page = FastDiv::of(out_page_size);
  a.B = (int)B, a.H = (int)Hkv, a.cap = (int)(n_table * page_size), a.budget = (int)budget, a.recent = (int)recent;
  a.row16 = FastDiv::of(row / 16);
  // parts that together fill the CUs once, of 64 rows at least (with 512 in all the
  // larger case above takes 48 us: a second choice for every CU); one where the
  // weights move in place, as the others would still be reading them
  int64_t parts = 256 / (B * Hkv);
  if (parts > (budget + 63) / 64) parts = (budget + 63) / 64;
  if (parts < 1 || (weights_out && weights_out == weights)) parts = 1;
  a.parts = (int)parts, a.clear = clear_behind != 0;
  const dim3 grid((uint32_t)(B * Hkv * parts));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.cap <= NT * kRegs)
    evict_kernel<true><<<grid, dim3(NT), 0, st>>>(a);
  else
    evict_kernel<false><<<grid, dim3(NT), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}
