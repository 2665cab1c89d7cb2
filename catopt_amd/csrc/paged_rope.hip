// RMS norm of each head of q and k and their position rotation in one pass,
// the keys and values going to the cache's pages where slots are given.
//
//   y = x rsqrt(mean(x^2) + eps) w;  (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// HBM bounds it: each row is read once and written once.
//
// The vector kernel gives a head L lanes, each with two 16-byte pieces of the
// row that rotate with each other: pieces i and i + rot / 2 further on, or two
// neighbours where the pairs are.  So a lane rotates what it holds, the norm's
// sum is the only exchange, and one load of its cos and sin serves every head
// of the token that the wave works on.  Any other layout takes the kernel with
// a wave per head, whose pairs meet in LDS.
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
  int64_t N, n_pos, ld_table, n_slots;
  FastDiv page;
  int Hq, Hkv, heads, d, rot, pairs;
  float eps;
};

// Where token n's key and value go: its slot's page (-1: outside the pages,
// nothing is written) and place in it.
struct Slot {
  int64_t page;
  int off;
};
__device__ __forceinline__ Slot slot_of(const RopeArgs& a, int64_t n) {
  Slot r{-1, 0};
  if (!a.slots) return r;
  const int64_t s = a.slots[n];
  if (s < 0 || s >= a.n_slots) return r;
  r.page = a.page.div((uint32_t)s);
  r.off = (int)((uint32_t)s - (uint32_t)r.page * a.page.d);
  return r;
}

// The row that (token, head) reads and the one it writes (null: none).  Heads:
// Hq of q, Hkv of k, then Hkv of v.
template <typename T>
__device__ __forceinline__ void rows_of(const RopeArgs& a, int64_t n, int h, const Slot& slot, const T*& src, T*& dst) {
  if (h < a.Hq) {
    src = static_cast<const T*>(a.q) + n * a.q_st + h * a.q_sh;
    dst = static_cast<T*>(a.q_out) + (n * a.Hq + h) * a.d;
    return;
  }
  h -= a.Hq;
  const bool value = h >= a.Hkv;
  if (value) h -= a.Hkv;
  src = value ? static_cast<const T*>(a.v) + n * a.v_st + h * a.v_sh : static_cast<const T*>(a.k) + n * a.k_st + h * a.k_sh;
  if (!a.slots)
    dst = static_cast<T*>(a.k_out) + (n * a.Hkv + h) * a.d;
  else if (slot.page < 0)
    dst = nullptr;
  else
    dst = value ? static_cast<T*>(a.v_out) + slot.page * a.vo_p + h * a.vo_h + slot.off * a.vo_s
                : static_cast<T*>(a.k_out) + slot.page * a.ko_p + h * a.ko_h + slot.off * a.ko_s;
}

constexpr int kMaxD = 256;

// One wave per (token, head): any head dim up to 256, any rotation.
template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_any(RopeArgs a) {
  __shared__ float rows[4][kMaxD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t unit = blockIdx.x * 4 + wave;  // below 2^26
  const bool live = unit < (uint64_t)a.N * a.heads;
  const int64_t n = live ? unit / (uint32_t)a.heads : 0;
  const int h = live ? (int)(unit - (uint32_t)n * a.heads) : 0;
  const T* src;
  T* dst;
  rows_of<T>(a, n, h, slot_of(a, n), src, dst);
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

// Elements of a 16-byte piece.
template <typename T>
constexpr int kPiece = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const u32x4& w, float* f) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
}

template <typename T>
__device__ __forceinline__ u32x4 pack(const float* f) {
  if constexpr (sizeof(T) == 2)
    return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  else
    return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
}

// Rows that together pass the 256 MB of the memory-side cache gain nothing from
// staying in the caches, and cost what does (16384 tokens of 96 heads, 814 MB:
// 156 -> 149 us); fewer ones are left there for the attention that reads them.
template <bool ONCE>
__device__ __forceinline__ u32x4 load_piece(const void* p) {
  const u32x4* x = static_cast<const u32x4*>(p);
  return ONCE ? __builtin_nontemporal_load(x) : *x;
}
template <bool ONCE>
__device__ __forceinline__ void store_piece(void* p, u32x4 w) {
  u32x4* x = static_cast<u32x4*>(p);
  if (ONCE)
    __builtin_nontemporal_store(w, x);
  else
    *x = w;
}

// A wave works on `rounds` times 64 / L heads of one token, one round after the
// other: eight waves to a SIMD hide the loads.
template <typename T, int L, bool ONCE>
__global__ __launch_bounds__(256) void qk_norm_rope_vec(RopeArgs a, FastDiv groups, int rounds) {
  constexpr int E = kPiece<T>, HPW = 64 / L;
  const int lane = threadIdx.x & 63, sub = lane % L, hs = lane / L;
  const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // below 2^26
  const int64_t n = groups.div(unit);
  if (n >= a.N) return;
  const int h0 = (int)(unit - (uint32_t)n * groups.d) * rounds * HPW + hs;
  const int pieces = a.d / E, turning = a.rot / (2 * E);  // lanes sub < turning rotate
  int c0, c1;
  if (!a.pairs && sub < turning) {
    c0 = sub, c1 = sub + turning;
  } else {
    c0 = a.pairs ? 2 * sub : 2 * turning + 2 * (sub - turning), c1 = c0 + 1;
  }
  const bool has0 = c0 < pieces, has1 = c1 < pieces;
  const Slot slot = slot_of(a, n);
  float cs[E], sn[E];
  if (sub < turning) {
    const int64_t p = a.pos[n];
    const bool known = p >= 0 && p < a.n_pos;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const int64_t at = (known ? p : 0) * a.ld_table + sub * E + i;
      f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f}, s = c;
      if (known) {
        c = *reinterpret_cast<const f32x4*>(a.cos + at);
        s = *reinterpret_cast<const f32x4*>(a.sin + at);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cs[i + j] = known ? c[j] : __builtin_nanf("");
        sn[i + j] = known ? s[j] : __builtin_nanf("");
      }
    }
  }
  for (int u = 0; u < rounds; ++u) {
    const int h = h0 + u * HPW;
    if (h >= a.heads) break;
    const T* src;
    T* dst;
    rows_of<T>(a, n, h, slot, src, dst);
    u32x4 x0 = u32x4{0, 0, 0, 0}, x1 = x0;
    if (has0) x0 = load_piece<ONCE>(src + c0 * E);
    if (has1) x1 = load_piece<ONCE>(src + c1 * E);
    if (h < a.Hq + a.Hkv) {  // else a value, stored as it is
      const T* w = static_cast<const T*>(h < a.Hq ? a.qw : a.kw);
      float f[2][E];
      unpack<T>(x0, f[0]);
      unpack<T>(x1, f[1]);
      if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) ss += f[0][i] * f[0][i] + f[1][i] * f[1][i];
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);  // within a head's lanes
        const float r = rsqrtf(ss / (float)a.d + a.eps);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          u32x4 ww = u32x4{0, 0, 0, 0};
          if (k ? has1 : has0) ww = *reinterpret_cast<const u32x4*>(w + (k ? c1 : c0) * E);
          float wf[E];
          unpack<T>(ww, wf);
#pragma unroll
          for (int i = 0; i < E; ++i) f[k][i] *= r * wf[i];
        }
      }
      if (sub < turning) {
        if (a.pairs) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < E; i += 2) {
              const float c = cs[(k * E + i) / 2], s = sn[(k * E + i) / 2], p = f[k][i], q = f[k][i + 1];
              f[k][i] = p * c - q * s;
              f[k][i + 1] = q * c + p * s;
            }
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const float p = f[0][i], q = f[1][i];
            f[0][i] = p * cs[i] - q * sn[i];
            f[1][i] = q * cs[i] + p * sn[i];
          }
        }
      }
      x0 = pack<T>(f[0]);
      x1 = pack<T>(f[1]);
    }
    if (dst && has0) store_piece<ONCE>(dst + c0 * E, x0);
    if (dst && has1) store_piece<ONCE>(dst + c1 * E, x1);
  }
}

// Whether every row is made of 16-byte pieces that the rotation pairs whole.
template <typename T>
bool in_pieces(const RopeArgs& a) {
  constexpr int E = kPiece<T>;
  const int64_t s[] = {a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh, a.ko_p, a.ko_h, a.ko_s, a.vo_p, a.vo_h, a.vo_s};
  for (int64_t x : s)
    if (x % E) return false;
  for (const void* p : {a.q, a.k, a.v, a.qw, a.kw, (const void*)a.cos, (const void*)a.sin, (const void*)a.q_out,
                        (const void*)a.k_out, (const void*)a.v_out})
    if (!aligned16(p)) return false;
  return a.d % E == 0 && a.rot % (2 * E) == 0 && a.ld_table % 4 == 0;
}

template <typename T, int L>
int32_t launch_vec(const RopeArgs& a, hipStream_t s) {
  constexpr int HPW = 64 / L;
  // a wave takes four rounds of heads where that leaves four waves to a SIMD
  const int64_t all = (a.heads + HPW - 1) / HPW;
  const int rounds = a.N * ((all + 3) / 4) >= 4096 ? 4 : 1;
  const int64_t groups = (all + rounds - 1) / rounds, blocks = (a.N * groups + 3) / 4;
  if (!grid_fits(blocks, 256)) return CATOPT_E_UNSUPPORTED;
  const bool once = 2 * a.N * a.heads * a.d * (int64_t)sizeof(T) > (256LL << 20);
  if (once)
    qk_norm_rope_vec<T, L, true><<<dim3((uint32_t)blocks), dim3(256), 0, s>>>(a, FastDiv::of(groups), rounds);
  else
    qk_norm_rope_vec<T, L, false><<<dim3((uint32_t)blocks), dim3(256), 0, s>>>(a, FastDiv::of(groups), rounds);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

template <typename T>
int32_t launch(const RopeArgs& a, hipStream_t s) {
  if (in_pieces<T>(a)) {
    const int lanes = (a.d / kPiece<T> + 1) / 2;  // of a head
    if (lanes <= 4) return launch_vec<T, 4>(a, s);
    if (lanes <= 8) return launch_vec<T, 8>(a, s);
    if (lanes <= 16 || sizeof(T) == 2) return launch_vec<T, 16>(a, s);
    if constexpr (sizeof(T) == 4) return launch_vec<T, 32>(a, s);
  }
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
  if (!strides || !positions || (Hq && (!q || !q_out)) || (Hkv && (!k || (!k_out && !(slots && n_pages == 0)))))
    return CATOPT_E_INVAL;
  if (rot > 0 && n_pos > 0 && (!cos || !sin || ld_table < rot / 2)) return CATOPT_E_INVAL;
  if (slots && ((Hkv && (!v || (n_pages > 0 && !v_out))) || n_pages < 0 || page_size < 1)) return CATOPT_E_INVAL;
  const int64_t np = slots ? n_pages : 0, ns = slots ? page_size : 0, nv = slots ? N : 0;
  const Strides st(strides, {N, Hq, N, Hkv, nv, Hkv, np, Hkv, ns, np, Hkv, ns}, 1);
  if (!st.fit) return CATOPT_E_INVAL;
  if (slots) {
    if (n_pages > (1LL << 31) || page_size > (1LL << 31) || n_pages * page_size >= (1LL << 31)) return CATOPT_E_UNSUPPORTED;
    const int64_t size = dtype == CATOPT_BF16 ? 2 : 4;
    const Layout lk = layout_pages(k_out, size, n_pages, Hkv, page_size, d, st.s + 6);
    const Layout lv = layout_pages(v_out, size, n_pages, Hkv, page_size, d, st.s + 9);
    const Layout in[3] = {layout3(q, size, N, st.s[0], Hq, st.s[1], d), layout3(k, size, N, st.s[2], Hkv, st.s[3], d),
                          layout3(v, size, N, st.s[4], Hkv, st.s[5], d)};
    // keys and values may be parts of one storage, so their ranges may interleave
    if (lk.folded() || lv.folded() || (k_out == v_out && !lk.empty())) return CATOPT_E_INVAL;
    for (const Layout& x : in)
      if (lk.overlaps(x) || lv.overlaps(x)) return CATOPT_E_INVAL;
  }
  RopeArgs a{};
  a.q = q, a.k = k, a.v = v, a.qw = q_weight, a.kw = k_weight;
  a.cos = cos, a.sin = sin, a.pos = positions, a.slots = slots;
  a.q_out = q_out, a.k_out = k_out, a.v_out = v_out;
  a.q_st = st.s[0], a.q_sh = st.s[1], a.k_st = st.s[2], a.k_sh = st.s[3];
  if (slots) {
    a.v_st = st.s[4], a.v_sh = st.s[5];
    a.ko_p = st.s[6], a.ko_h = st.s[7], a.ko_s = st.s[8];
    a.vo_p = st.s[9], a.vo_h = st.s[10], a.vo_s = st.s[11];
  }
  a.N = N, a.n_pos = n_pos, a.ld_table = ld_table;
  a.n_slots = slots ? n_pages * page_size : 0;
  a.page = FastDiv::of(slots ? page_size : 1);
  a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.heads = (int)(Hq + (slots ? 2 : 1) * Hkv);
  a.d = (int)d, a.rot = (int)rot, a.pairs = interleaved != 0, a.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == CATOPT_BF16 ? launch<uint16_t>(a, s) : launch<float>(a, s);
}
