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

// One workgroup per (sequence, head).  Radix select over 8 bits at a time
// finds the rank of the last key that stays and how many of its equals do
// (the first ones); one pass in key order then lists the kept keys.
__global__ __launch_bounds__(NT) void evict_select(EvictArgs a) {
  __shared__ uint32_t hist[256], sh_bin, sh_left, wave_sum[2][NT / 64];
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = min(max(a.lens[b], 0), a.cap), m = min(n, a.budget);
  const int old = n - min(a.recent, m);  // keys from here on stay
  const float* w = a.w + b * a.w_b + h * a.w_h;
  float* w_out = a.w_out ? a.w_out + b * a.wo_b + h * a.wo_h : nullptr;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = m;
  uint32_t need = (uint32_t)(m - (n - old)), prefix = 0;  // of the first `old` keys, `need` stay
  if (need > 0 && need < (uint32_t)old) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int j = tid; j < old; j += NT) {
        const uint32_t r = rank_of(w[j]);
        if ((r & mask) == prefix) atomicAdd(&hist[(r >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = need;
        int bin = 255;
        while (bin > 0 && hist[bin] < left) left -= hist[bin--];
        sh_bin = (uint32_t)bin;
        sh_left = left;
      }
      __syncthreads();
      prefix |= sh_bin << shift;
      need = sh_left;
      __syncthreads();
    }
  } else if (need > 0) {
    need = 0, prefix = 0;  // every old key stays: every rank is at least 0
  } else {
    prefix = 0xffffffffu;  // none does
  }
  // keys above the last rank stay, and the first `need` of that rank itself
  // (all of them where every old key stays)
  const bool all = m - (n - old) == old, none = m == n - old;
  uint32_t base = 0, base_eq = 0;
  for (int j0 = 0; j0 < n; j0 += NT) {
    const int j = j0 + tid;
    const float wj = j < n ? w[j] : 0.f;
    const uint32_t r = rank_of(wj);
    const bool is_old = j < old;
    const bool above = j < n && (!is_old || all || (!none && r > prefix));
    const bool equal = is_old && !all && !none && r == prefix;
    const uint64_t below = (1ull << lane) - 1, be = __ballot(equal);
    if (lane == 0) wave_sum[0][wave] = __popcll(be);
    __syncthreads();
    uint32_t eq_before = base_eq + __popcll(be & below), eq_total = 0;
    for (int i = 0; i < NT / 64; ++i) {
      if (i < wave) eq_before += wave_sum[0][i];
      eq_total += wave_sum[0][i];
    }
    const bool stay = above || (equal && eq_before < need);
    const uint64_t bs = __ballot(stay);
    if (lane == 0) wave_sum[1][wave] = __popcll(bs);
    __syncthreads();
    uint32_t at = base + __popcll(bs & below), total = 0;
    for (int i = 0; i < NT / 64; ++i) {
      if (i < wave) at += wave_sum[1][i];
      total += wave_sum[1][i];
    }
    if (stay && at < (uint32_t)m) {
      kept[at] = j;
      if (w_out) w_out[at] = wj;  // at <= j, and every weight up to j0 + NT has been read
    }
    base += total;
    base_eq += eq_total;
    __syncthreads();
  }
  for (int j = m + tid; j < a.budget; j += NT) kept[j] = -1;
}

// 16 bytes of one kept row of k and of v per thread.
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
    k = static_cast<const u32x4*>(a.k.p)[from * a.k.s_page + h * a.k.s_head + si * a.k.s_slot + piece];
    v = static_cast<const u32x4*>(a.v.p)[from * a.v.s_page + h * a.v.s_head + si * a.v.s_slot + piece];
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
  if (n_table * page_size > lim) return CATOPT_E_UNSUPPORTED;
  if (n_out_table * out_page_size < budget) return CATOPT_E_INVAL;
  if (B == 0) return CATOPT_OK;
  const int64_t step = 16 / (dtype == CATOPT_BF16 ? 2 : 4);
  if (!strides || !strides_fit(strides, 12, step) || !strides_fit(strides + 12, 4, 1)) return CATOPT_E_INVAL;
  if (!kv_lens || !kept || !new_lens || !out_table || (n_table > 0 && (!block_table || !weights))) return CATOPT_E_INVAL;
  if ((n_pages > 0 && (!k_pages || !v_pages)) || (n_out_pages > 0 && (!k_out || !v_out))) return CATOPT_E_INVAL;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out)) return CATOPT_E_INVAL;
  EvictArgs a{};
  const int64_t* s = strides;
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
  if (!grid_fits(B * Hkv, NT)) return CATOPT_E_UNSUPPORTED;  // so B Hkv < 2^22 and the product below < 2^62
  const int64_t blocks = (B * Hkv * budget * a.row16 + 255) / 256;
  if (!grid_fits(blocks, 256)) return CATOPT_E_UNSUPPORTED;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  evict_select<<<dim3((uint32_t)(B * Hkv)), dim3(NT), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  evict_move<<<dim3((uint32_t)blocks), dim3(256), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}
