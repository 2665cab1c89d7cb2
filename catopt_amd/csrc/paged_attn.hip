// Attention of each sequence's new tokens over its paged cache, and the sum of
// every key's attention weight.
//
// One workgroup per (token, query head): its lanes take one key each, the row's
// softmax statistics meet in LDS, and each thread then adds one column of the
// values.  The weights follow in a second launch, one thread per key.
#include "paged.hpp"

namespace catopt {
namespace {

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  int64_t q_t, q_h, k_p, k_h, k_s, v_p, v_h, v_s, o_t, o_h, wi_b, wi_h, wo_b, wo_h;
  const int32_t *table, *lens, *starts;
  int64_t table_ld, n_pages, N;
  float *m_out, *l_out, *w_out, *stats;
  const float* w_in;
  FastDiv page;
  int B, Hq, Hkv, G, d, cap, normalize, causal;
  float scale;
};

constexpr int NT = 256;
constexpr float kNegInf = -__builtin_inff();

// The sequence of row n, its rows and its keys; -1 behind the last sequence.
__device__ __forceinline__ int seq_of(const PagedArgs& a, int64_t n, int& row0, int& nq, int& len) {
  for (int b = 0; b < a.B; ++b) {
    seq_rows(a.starts, b, a.N, row0, nq);
    if (row0 <= n && n < row0 + nq) {
      len = min(max(a.lens[b], 0), a.cap);
      return b;
    }
  }
  return -1;
}

// q . k of one key, -inf where its page is invalid
__device__ __forceinline__ float score(const PagedArgs& a, const uint16_t* q, int b, int h, int j) {
  const uint32_t tp = a.page.div(j);
  const int64_t page = a.table[b * a.table_ld + tp];
  if (page < 0 || page >= a.n_pages) return kNegInf;
  const uint16_t* k = a.k + page * a.k_p + h * a.k_h + (int64_t)(j - tp * a.page.d) * a.k_s;
  float s = 0.f;
  for (int e = 0; e < a.d; ++e) s += bf16_to_f32(q[e]) * bf16_to_f32(k[e]);
  return s * a.scale;
}

__global__ __launch_bounds__(NT) void paged_attn_rows(PagedArgs a) {
  __shared__ float red[NT], p[NT];
  const int64_t n = blockIdx.x / a.Hq;
  const int hq = blockIdx.x - (int)(n * a.Hq), h = hq / a.G, tid = threadIdx.x;
  int row0, nq, len;
  const int b = seq_of(a, n, row0, nq, len);
  if (b < 0) return;
  const int64_t lim = a.causal ? (int64_t)len - nq + (n - row0) : (int64_t)len - 1;  // last key seen
  const int end = lim < 0 ? 0 : (int)(lim + 1 < len ? lim + 1 : len);
  const uint16_t* q = a.q + n * a.q_t + hq * a.q_h;
  float m = kNegInf, l = 0.f, acc = 0.f;
  for (int j0 = 0; j0 < end; j0 += NT) {
    const int j = j0 + tid;
    const float s = j < end ? score(a, q, b, h, j) : kNegInf;
    red[tid] = s;
    __syncthreads();
    float mx = m;
    for (int i = 0; i < NT; ++i) mx = fmaxf(mx, red[i]);
    const float old = m == kNegInf ? 0.f : __expf(m - mx);
    p[tid] = s == kNegInf ? 0.f : __expf(s - mx);
    __syncthreads();
    m = mx;
    l *= old;
    acc *= old;
    for (int i = 0; i < NT && j0 + i < end; ++i) {
      const int64_t page = a.table[b * a.table_ld + a.page.div(j0 + i)];
      l += p[i];
      if (tid < a.d && page >= 0 && page < a.n_pages) {
        const uint32_t slot = (j0 + i) - a.page.div(j0 + i) * a.page.d;
        acc += p[i] * bf16_to_f32(a.v[page * a.v_p + h * a.v_h + slot * a.v_s + tid]);
      }
    }
    __syncthreads();
  }
  if (tid < a.d) {
    const float x = l == 0.f ? (a.normalize == 2 ? 0.f : __builtin_nanf("")) : acc / l;
    a.o[n * a.o_t + hq * a.o_h + tid] = f32_to_bf16(x);
  }
  if (tid == 0) {
    if (a.m_out) a.m_out[n * a.Hq + hq] = m;
    if (a.l_out) a.l_out[n * a.Hq + hq] = l;
    if (a.stats) {
      a.stats[2 * (n * a.Hq + hq)] = m;
      a.stats[2 * (n * a.Hq + hq) + 1] = l;
    }
  }
}

__global__ __launch_bounds__(NT) void paged_attn_weights(PagedArgs a, int blocks) {
  const int bh = blockIdx.x / blocks, b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int j = (blockIdx.x - bh * blocks) * NT + threadIdx.x;
  int row0, nq;
  seq_rows(a.starts, b, a.N, row0, nq);
  const int len = min(max(a.lens[b], 0), a.cap);
  if (j >= len) return;
  float w = 0.f;
  for (int i = 0; i < nq; ++i) {
    if (a.causal && j > len - nq + i) continue;
    for (int g = 0; g < a.G; ++g) {
      const int64_t n = row0 + i, hq = h * a.G + g;
      const float m = a.stats[2 * (n * a.Hq + hq)], l = a.stats[2 * (n * a.Hq + hq) + 1];
      if (l == 0.f) continue;
      w += __expf(score(a, a.q + n * a.q_t + hq * a.q_h, b, h, j) - m) / l;
    }
  }
  if (a.w_in && j < len - nq) w += a.w_in[b * a.wi_b + h * a.wi_h + j];
  a.w_out[b * a.wo_b + h * a.wo_h + j] = w;
}

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int64_t catopt_hip_paged_attn_workspace_bytes(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d,
                                                         int64_t n_table, int64_t page_size, int32_t weights) {
  const int64_t lim = 1LL << 30;
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || d < 8 || d > 128 || d % 8) return -1;
  if (n_table < 0 || page_size < 8 || page_size % 8) return -1;
  if (B > lim || N > lim || Hq > 65535 || n_table > lim || page_size > lim || n_table * page_size > lim) return -1;
  return weights ? 8 * N * Hq : 0;
}

extern "C" int32_t catopt_hip_paged_attn_fwd(
    int32_t dtype, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d, const void* q, const void* k_pages,
    const void* v_pages, int64_t n_pages, int64_t page_size, const int32_t* block_table, int64_t table_ld,
    int64_t n_table, const int32_t* kv_lens, const int32_t* q_starts, float scale, int32_t causal, int32_t normalize,
    void* o, float* m_out, float* l_out, const float* weights_in, float* weights_out, const int64_t* strides,
    void* workspace, int64_t workspace_bytes, void* stream) {
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || n_pages < 0 || n_table < 0 || page_size < 1 || table_ld < 0)
    return CATOPT_E_INVAL;
  if (normalize < 1 || normalize > 2) return CATOPT_E_INVAL;
  if (dtype != CATOPT_BF16 || d < 8 || d > 128 || d % 8 || page_size % 8) return CATOPT_E_UNSUPPORTED;
  if (!(scale > 0.f) || !__builtin_isfinite(scale)) return CATOPT_E_UNSUPPORTED;
  const int64_t need = catopt_hip_paged_attn_workspace_bytes(B, N, Hq, Hkv, d, n_table, page_size, weights_out != nullptr);
  if (need < 0) return CATOPT_E_UNSUPPORTED;
  if (B == 0 || N == 0) return CATOPT_OK;
  if (!q || !o || !kv_lens || !q_starts || !strides || (n_table > 0 && !block_table)) return CATOPT_E_INVAL;
  if (n_pages > 0 && (!k_pages || !v_pages)) return CATOPT_E_INVAL;
  if (!strides_fit(strides, 10, 8) || !strides_fit(strides + 10, 4, 1)) return CATOPT_E_INVAL;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o)) return CATOPT_E_INVAL;
  if (weights_in && !weights_out) return CATOPT_E_INVAL;
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return CATOPT_E_WORKSPACE;
  PagedArgs a{};
  const int64_t* s = strides;
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k_pages);
  a.v = static_cast<const uint16_t*>(v_pages), a.o = static_cast<uint16_t*>(o);
  a.q_t = s[0], a.q_h = s[1], a.k_p = s[2], a.k_h = s[3], a.k_s = s[4], a.v_p = s[5], a.v_h = s[6], a.v_s = s[7];
  a.o_t = s[8], a.o_h = s[9], a.wi_b = s[10], a.wi_h = s[11], a.wo_b = s[12], a.wo_h = s[13];
  a.table = block_table, a.lens = kv_lens, a.starts = q_starts, a.table_ld = table_ld, a.n_pages = n_pages, a.N = N;
  a.m_out = m_out, a.l_out = l_out, a.w_in = weights_in, a.w_out = weights_out;
  a.stats = weights_out ? static_cast<float*>(workspace) : nullptr;
  a.page = FastDiv::of(page_size);
  a.B = (int)B, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.d = (int)d, a.cap = (int)(n_table * page_size);
  a.normalize = normalize, a.causal = causal != 0, a.scale = scale;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (!grid_fits(N * Hq, NT)) return CATOPT_E_UNSUPPORTED;
  paged_attn_rows<<<dim3((uint32_t)(N * Hq)), dim3(NT), 0, st>>>(a);
  CATOPT_LAUNCH_CHECK();
  if (weights_out && a.cap > 0) {
    const int64_t blocks = (a.cap + NT - 1) / NT;
    if (!grid_fits(B * Hkv * blocks, NT)) return CATOPT_E_UNSUPPORTED;
    paged_attn_weights<<<dim3((uint32_t)(B * Hkv * blocks)), dim3(NT), 0, st>>>(a, (int)blocks);
    CATOPT_LAUNCH_CHECK();
  }
  return CATOPT_OK;
}
