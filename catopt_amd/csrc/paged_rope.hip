// RMS norm of each head of q and k and their position rotation in one pass,
// the keys and values going to the cache's pages where slots are given.
//
//   y = x rsqrt(mean(x^2) + eps) w;  (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// HBM bounds it: each row is read once and written once.
#include "paged.hpp"

namespace catopt {
namespace {

struct RopeArgs {
  const void *q, *k, *v, *qw, *kw;
  const float *cos, *sin;
  const int64_t *pos, *slots;
  void *q_out, *k_out, *v_out;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;          // token, head
  int64_t ko_p, ko_h, ko_s, vo_p, vo_h, vo_s;          // page, head, slot
  int64_t N, n_pos, ld_table, n_pages, page_size;
  int Hq, Hkv, heads, d, rot, pairs;
  float eps;
};

// The row that (token, head) reads and the one it writes (null: a slot
// outside the pages).  Heads: Hq of q, Hkv of k, then Hkv of v.
template <typename T>
__device__ __forceinline__ void rows_of(const RopeArgs& a, int64_t n, int h, const T*& src, T*& dst) {
  if (h < a.Hq) {
    src = static_cast<const T*>(a.q) + n * a.q_st + h * a.q_sh;
    dst = static_cast<T*>(a.q_out) + (n * a.Hq + h) * a.d;
    return;
  }
  h -= a.Hq;
  const bool value = h >= a.Hkv;
  if (value) h -= a.Hkv;
  src = value ? static_cast<const T*>(a.v) + n * a.v_st + h * a.v_sh : static_cast<const T*>(a.k) + n * a.k_st + h * a.k_sh;
  if (!a.slots) {
    dst = static_cast<T*>(a.k_out) + (n * a.Hkv + h) * a.d;
    return;
  }
  const int64_t slot = a.slots[n];
  const int64_t page = slot < 0 ? -1 : slot / a.page_size;
  if (page < 0 || page >= a.n_pages) {
    dst = nullptr;
    return;
  }
  const int64_t off = slot - page * a.page_size;
  dst = value ? static_cast<T*>(a.v_out) + page * a.vo_p + h * a.vo_h + off * a.vo_s
              : static_cast<T*>(a.k_out) + page * a.ko_p + h * a.ko_h + off * a.ko_s;
}

constexpr int kMaxD = 256;

// One wave per (token, head): any head dim up to 256, any rotation.
template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_any(RopeArgs a) {
  __shared__ float rows[4][kMaxD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const bool live = unit < a.N * a.heads;
  const int64_t n = live ? unit / a.heads : 0;
  const int h = live ? (int)(unit - n * a.heads) : 0;
  const T* src;
  T* dst;
  rows_of<T>(a, n, h, src, dst);
  const bool value = h >= a.Hq + a.Hkv;
  const T* w = static_cast<const T*>(value ? nullptr : h < a.Hq ? a.qw : a.kw);
  float x[kMaxD / 64], ss = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxD / 64; ++i) {
    const int e = lane + 64 * i;
    x[i] = live && e < a.d ? load_f32(src, e) : 0.f;
    ss += x[i] * x[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
  const float r = w ? rsqrtf(ss / (float)a.d + a.eps) : 1.f;
#pragma unroll
  for (int i = 0; i < kMaxD / 64; ++i) {
    const int e = lane + 64 * i;
    if (e < a.d) {
      if (w) x[i] *= r * load_f32(w, e);
      rows[wave][e] = x[i];
    }
  }
  __syncthreads();
  if (!live || !dst) return;
  const int64_t p = value ? 0 : a.pos[n];
  const bool known = p >= 0 && p < a.n_pos;
  const int half = a.rot / 2;
#pragma unroll
  for (int i = 0; i < kMaxD / 64; ++i) {
    const int e = lane + 64 * i;
    if (e >= a.d) continue;
    float y = x[i];
    if (!value && e < a.rot) {
      const bool second = a.pairs ? e & 1 : e >= half;
      const int f = a.pairs ? e >> 1 : second ? e - half : e;
      const int other = a.pairs ? e ^ 1 : second ? e - half : e + half;
      const float c = known ? a.cos[p * a.ld_table + f] : __builtin_nanf("");
      const float s = known ? a.sin[p * a.ld_table + f] : __builtin_nanf("");
      const float z = rows[wave][other];
      y = second ? y * c + z * s : y * c - z * s;
    }
    store_f32(dst, e, y);
  }
}

template <typename T>
int32_t launch(const RopeArgs& a, hipStream_t s) {
  const int64_t blocks = (a.N * a.heads + 3) / 4;
  if (!grid_fits(blocks, 256)) return CATOPT_E_UNSUPPORTED;
  qk_norm_rope_any<T><<<dim3((uint32_t)blocks), dim3(256), 0, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int32_t catopt_hip_qk_norm_rope(int32_t dtype, int64_t N, int64_t Hq, int64_t Hkv, int64_t d, int64_t rot,
                                           int32_t interleaved, const void* q, const void* k, const void* v,
                                           const void* q_weight, const void* k_weight, float eps, const float* cos,
                                           const float* sin, int64_t n_pos, int64_t ld_table,
                                           const int64_t* positions, void* q_out, void* k_out, void* v_out,
                                           const int64_t* strides, const int64_t* slots, int64_t n_pages,
                                           int64_t page_size, void* stream) {
  if (N < 0 || Hq < 0 || Hkv < 0 || d < 1 || rot < 0 || rot > d || rot % 2 || n_pos < 0) return CATOPT_E_INVAL;
  if (dtype != CATOPT_F32 && dtype != CATOPT_BF16) return CATOPT_E_UNSUPPORTED;
  if (d > kMaxD || Hq > (1 << 20) || Hkv > (1 << 20) || N > (1LL << 40)) return CATOPT_E_UNSUPPORTED;
  if (N == 0 || Hq + Hkv == 0) return CATOPT_OK;
  if (!strides || !positions || (Hq && (!q || !q_out)) || (Hkv && (!k || !k_out))) return CATOPT_E_INVAL;
  if (rot > 0 && n_pos > 0 && (!cos || !sin || ld_table < rot / 2)) return CATOPT_E_INVAL;
  const int n_strides = slots ? 12 : 4;
  if (!strides_fit(strides, n_strides, 1)) return CATOPT_E_INVAL;
  if (slots && ((Hkv && (!v || !v_out)) || n_pages < 0 || page_size < 1)) return CATOPT_E_INVAL;
  RopeArgs a{};
  a.q = q, a.k = k, a.v = v, a.qw = q_weight, a.kw = k_weight;
  a.cos = cos, a.sin = sin, a.pos = positions, a.slots = slots;
  a.q_out = q_out, a.k_out = k_out, a.v_out = v_out;
  a.q_st = strides[0], a.q_sh = strides[1], a.k_st = strides[2], a.k_sh = strides[3];
  if (slots) {
    a.v_st = strides[4], a.v_sh = strides[5];
    a.ko_p = strides[6], a.ko_h = strides[7], a.ko_s = strides[8];
    a.vo_p = strides[9], a.vo_h = strides[10], a.vo_s = strides[11];
  }
  a.N = N, a.n_pos = n_pos, a.ld_table = ld_table, a.n_pages = n_pages, a.page_size = page_size;
  a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.heads = (int)(Hq + (slots ? 2 : 1) * Hkv);
  a.d = (int)d, a.rot = (int)rot, a.pairs = interleaved != 0, a.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == CATOPT_BF16 ? launch<uint16_t>(a, s) : launch<float>(a, s);
}
