// What the paged attention kernels share: a call's arguments, the tiles of
// query rows, the page reads, the products and the split keys' bookkeeping.
#pragma once
#include "attention.hpp"
#include "paged.hpp"

namespace catopt {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  int64_t q_t, q_h, k_p, k_h, k_s, v_p, v_h, v_s, o_t, o_h, wi_b, wi_h, wo_b, wo_h;
  const int32_t *table, *lens, *starts;
  int64_t table_ld, n_pages, N;
  float *m_out, *l_out;  // [N, Hq], optional
  float* row_log;        // [N, Hq] m + log l of the row in log2 units, +inf where it sees no key; for the weights
  float* part;           // split keys' carriers: [row][split] (m, l), then [row][split][D]; row = n Hq + hq
  float* scores;         // [row][cap] q . k of the keys that the row's tile sees, -inf where masked; optional
  const float* w_in;
  float* w_out;
  FastDiv page, group;  // by the page size, by the query heads of a key head
  FastDiv q_heads, k_heads, ranges;  // by Hq, Hkv, splits
  int B, Hq, Hkv, G, d, cap, normalize, causal;
  int splits, min_keys;  // key ranges per tile at most, keys of one at least
  float scale;
  // Of the calls over two sets of keys, a set's part:
  const int32_t* groups;  // the set's sequences are groups of the call's (NULL: they are those), their first ones
  int n_seq;              // the call's sequences
  int part_ld, part_first;  // of a row's carriers: all, and the set's first
};

// Query rows of one key head are its G query heads of every token, a token's
// heads next to each other: row r of a sequence is token r / G, head r % G.
// A tile is R such rows; the tiles of sequence b begin at tile
// floor(row0 G / R) + b, which leaves each sequence as many as it needs
// whatever the lengths are, so the grid depends on N and B alone.
inline int64_t paged_tiles(int64_t N, int64_t G, int64_t B, int64_t R) { return N * G / R + B; }

struct PagedTile {
  int b, row0, nq, len, r0, rows;  // sequence, its tokens and keys; the tile's first row and its rows (0: no such tile)
  int off;                         // token i sees keys <= off + i
  int kend;                        // keys that some row of the tile sees
  int keys;                        // of each of its key ranges
  bool split;                      // it has several
};

// What a tile's workgroup does: the rows of a call over one set of keys; a set's
// carriers of a call over two; such a call's rows over the first set and then, with
// the same accumulators, over the second (the groups then have one more at either
// end, of the sequences outside them, without keys).
enum Form { kRows, kCarriers, kBothSets };

// The rows of sequence b, or of group b of them.
template <Form F>
__device__ __forceinline__ void set_rows(const PagedArgs& a, int b, int& row0, int& nq) {
  if (F == kRows || !a.groups) return seq_rows(a.starts, b, a.N, row0, nq);
  const int n = (int)a.N;
  int first, next;
  if (F == kBothSets)
    first = b == 0 ? 0 : a.groups[b - 1], next = b == a.B - 1 ? a.n_seq : a.groups[b];
  else
    first = a.groups[b], next = a.groups[b + 1];
  row0 = min(max(a.starts[min(max(first, 0), a.n_seq)], 0), n);
  nq = max(min(max(a.starts[min(max(next, 0), a.n_seq)], 0), n) - row0, 0);
}
// Its keys.
template <Form F>
__device__ __forceinline__ int set_len(const PagedArgs& a, int b) {
  if (F == kBothSets && (b == 0 || b == a.B - 1)) return 0;
  return min(max(a.lens[F == kBothSets ? b - 1 : b], 0), a.cap);
}

// Lane i looks at sequence i (of 64 at a time), so that the search and the
// sequence's own numbers are one memory latency.
template <int R, Form F>
__device__ __forceinline__ PagedTile paged_tile(const PagedArgs& a, int t) {
  const int lane = threadIdx.x & 63;
  PagedTile x{};
  x.b = -1;
  int64_t first = 0;
  for (int c = 0; c < a.B; c += 64) {  // the last sequence whose first tile is not behind t
    const int i = c + lane;
    int row0 = 0, nq = 0, len = 0;
    bool le = false;
    if (i < a.B) {
      set_rows<F>(a, i, row0, nq);
      len = set_len<F>(a, i);
      le = (int64_t)row0 * a.G / R + i <= t;
    }
    const int n = __popcll(__ballot(le));
    if (n > 0) {
      x.b = c + n - 1;
      x.row0 = __builtin_amdgcn_readlane(row0, n - 1);
      x.nq = __builtin_amdgcn_readlane(nq, n - 1);
      x.len = __builtin_amdgcn_readlane(len, n - 1);
      first = (int64_t)x.row0 * a.G / R + x.b;
    }
    if (n < 64) break;
  }
  if (x.b < 0) return x;
  const int64_t rows = (int64_t)x.nq * a.G, r0 = (t - first) * R;
  x.r0 = (int)r0;
  x.rows = r0 >= 0 && r0 < rows ? (int)min((int64_t)R, rows - r0) : 0;  // r0 < 0: starts that do not ascend
  return x;
}

// The keys a tile of rows [r0, r0 + rows) sees, and how they are split: in
// ranges of at least min_keys and a multiple of 128 (whole stages of every
// kernel).
__device__ __forceinline__ void paged_ranges(const PagedArgs& a, PagedTile& x) {
  x.off = a.causal ? x.len - x.nq : 0x3fffffff;
  const int last = x.off + (int)a.group.div(x.r0 + x.rows - 1);  // below 2^31: both are below 2^30
  x.kend = last < 0 ? 0 : min(x.len, last + 1);
  x.keys = (max((int)a.ranges.div(x.kend + a.splits - 1), a.min_keys) + 127) & ~127;
  x.split = x.kend > x.keys;
}
// Whether range s of a tile has keys (the first is there in any case).
__device__ __forceinline__ bool has_range(const PagedTile& x, int s) { return s == 0 || (int64_t)s * x.keys < x.kend; }
// The ranges of a tile: 64 at most, so lane s looks at range s.
__device__ __forceinline__ int count_ranges(const PagedTile& x) { return __popcll(__ballot(has_range(x, threadIdx.x & 63))); }

// A workgroup's key head, its tile and key range: the heads next to each other,
// then the ranges.
__device__ __forceinline__ void decode_block(const PagedArgs& a, uint32_t block, int& h, int& tile, int& range) {
  const uint32_t ts = a.k_heads.div(block);
  h = (int)(block - ts * a.k_heads.d);
  tile = (int)a.ranges.div(ts);
  range = (int)(ts - (uint32_t)tile * a.ranges.d);
}

// Where range `split` of row i has its carrier, counted in carriers; and where
// their numerators begin.
template <Form F>
__device__ __forceinline__ int64_t part_at(const PagedArgs& a, int64_t i, int split) {
  return F == kCarriers ? i * a.part_ld + a.part_first + split : i * a.splits + split;
}
template <Form F>
__device__ __forceinline__ float* part_numerators(const PagedArgs& a) {
  return a.part + ((2 * a.N * a.Hq * (F == kCarriers ? a.part_ld : a.splits) + 3) & ~(int64_t)3);
}

// exp2((from - to) c), 0 for an empty `from`.
__device__ __forceinline__ float move_factor(float from, float to, float c) {
  return from == kNegInf ? 0.f : __builtin_amdgcn_exp2f((from - to) * c);
}

// A row of the result: numerator piece x of a row with sum l.
__device__ __forceinline__ float finish(float x, float l, int normalize) {
  if (l == 0.f) return normalize == 2 ? 0.f : __builtin_nanf("");
  return x * (1.0f / l);
}

// A finished row's statistics: max m (units of q . k) and sum l.  The max of the
// kernels passes a NaN score by, the sum does not (but it is NaN with +inf, too):
// the carrier's m is NaN then, or a part whose only scores are NaN would compose as
// an empty one.
__device__ __forceinline__ void row_stats(const PagedArgs& a, int64_t i, float m, float l) {
  if (a.m_out) a.m_out[i] = l != l && m < __builtin_inff() ? l : m * a.scale;
  if (a.l_out) a.l_out[i] = l;
  if (a.row_log) a.row_log[i] = l == 0.f ? __builtin_inff() : m * (a.scale * kLog2e) + __builtin_amdgcn_logf(l);
}

__device__ __forceinline__ void add_weight(const PagedArgs& a, int b, int h, int key, int old, float w) {
  if (a.w_in && key < old) w += a.w_in[b * a.wi_b + h * a.wi_h + key];
  a.w_out[b * a.wo_b + h * a.wo_h + key] = w;
}

// Where 8 keys (a lane's) lie: pages hold a multiple of 8 keys, so the rows of 8
// are in one, and one buffer resource over them serves all loads of them.  Its
// range ends behind the last key; for keys of an invalid page, or behind the
// last key, it is empty, so that they read as zeros.  The lanes work these out
// for many groups at once; a load takes its group's from the lane by readlane.
struct KeyGroup {
  uint32_t k_lo, k_hi, k_bytes, v_lo, v_hi, v_bytes;
};

__device__ __forceinline__ int group_page(const PagedArgs& a, const int32_t* table, int key, int len) {
  return key < len ? table[a.page.div(key)] : -1;
}

// `bad`: keys before `len` whose page is invalid.
__device__ __forceinline__ KeyGroup key_group(const PagedArgs& a, const uint16_t* kb, const uint16_t* vb, int page, int key,
                                              int len, bool& bad) {
  const bool real = key < len, ok = real && page >= 0 && page < a.n_pages;
  bad = real && !ok;
  const int64_t pg = ok ? page : 0, slot = ok ? key - (int)(a.page.div(key) * a.page.d) : 0;
  const int rows = min(len - key, 8);
  const uint64_t k = reinterpret_cast<uint64_t>(kb + pg * a.k_p + slot * a.k_s);
  const uint64_t v = reinterpret_cast<uint64_t>(vb + pg * a.v_p + slot * a.v_s);
  KeyGroup r;
  r.k_lo = (uint32_t)k, r.k_hi = (uint32_t)(k >> 32), r.v_lo = (uint32_t)v, r.v_hi = (uint32_t)(v >> 32);
  r.k_bytes = ok ? ((rows - 1) * (uint32_t)a.k_s + a.d) * 2u : 0u;
  r.v_bytes = ok ? ((rows - 1) * (uint32_t)a.v_s + a.d) * 2u : 0u;
  return r;
}

__device__ __forceinline__ u32x4 lane_rsrc(uint32_t lo, uint32_t hi, uint32_t bytes, int lane) {
  u32x4 r;
  r.x = __builtin_amdgcn_readlane(lo, lane);
  r.y = __builtin_amdgcn_readlane(hi, lane);
  r.z = __builtin_amdgcn_readlane(bytes, lane);
  r.w = 0x00020000;
  return r;
}
__device__ __forceinline__ u32x4 k_rsrc(const KeyGroup& x, int lane) { return lane_rsrc(x.k_lo, x.k_hi, x.k_bytes, lane); }
__device__ __forceinline__ u32x4 v_rsrc(const KeyGroup& x, int lane) { return lane_rsrc(x.v_lo, x.v_hi, x.v_bytes, lane); }

// Two direct loads of 1 KB of rows, to `lds` and `step` bytes behind, as dma_buf
// makes one, with the non-temporal hint: for rows that are read once.  The
// resources come out of lanes just before, and an SGPR that a lane read has
// written must not be read by a memory instruction for five wait states, which
// the compiler does not see in here: the move and s_nop 3 are those five for all.
__device__ __forceinline__ void dma_rows_once(u32x4 rsrc0, uint32_t off0, u32x4 rsrc1, uint32_t off1, uint32_t lds,
                                              uint32_t step) {
  const uint32_t to0 = __builtin_amdgcn_readfirstlane(lds), to1 = __builtin_amdgcn_readfirstlane(lds + step);
  asm volatile(
      "s_mov_b32 m0, %4\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds\n\t"
      "s_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen nt lds" ::"v"(off0),
      "s"(rsrc0), "v"(off1), "s"(rsrc1), "s"(to0), "s"(to1)
      : "m0", "memory");
}

// The same for two loads of K (to `k_lds` and `step` behind) and two of V, for rows
// that are read again.
__device__ __forceinline__ void dma_rows4(u32x4 k0, u32x4 k1, uint32_t k_off, uint32_t k_lds, u32x4 v0, u32x4 v1,
                                          uint32_t v_off, uint32_t v_lds, uint32_t step) {
  const uint32_t to = __builtin_amdgcn_readfirstlane(k_lds), vto = __builtin_amdgcn_readfirstlane(v_lds);
  asm volatile(
      "s_mov_b32 m0, %6\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds\n\t"
      "s_add_u32 m0, m0, %8\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %7\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %4, 0 offen lds\n\t"
      "s_add_u32 m0, m0, %8\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds" ::"v"(k_off),
      "v"(v_off), "s"(k0), "s"(k1), "s"(v0), "s"(v1), "s"(to), "s"(vto), "s"(step)
      : "m0", "scc", "memory");
}

// A lane's byte offset from its group's first row: row `row` of the 8, 16-byte
// piece `piece` of it; pieces past d lie outside every resource.
__device__ __forceinline__ uint32_t group_offset(int64_t s_slot, int row, int piece, int d) {
  return piece * 8 < d ? (uint32_t)(row * (int)s_slot + piece * 8) * 2u : 0x7ffffff0u;
}

// V^T fragments of 32 keys from an LDS tile: vf[2 db + u], keys 16 u + {4 (G /
// 2) + j / 4, 8 further} and d block 32 db + 16 (G % 2) + 4 (j % 4) for lane
// group G = lane / 16, j = lane % 16 (the order of the score accumulator).
template <int D>
__device__ __forceinline__ void read_v(const char* Vs, int key0, bf16x8* vf) {
  const int lane = threadIdx.x & 63, G = lane >> 4, jj = lane & 15;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = key0 + 16 * u + 4 * (G >> 1) + (jj >> 2);
      const int d = 32 * db + 16 * (G & 1) + 4 * (jj & 3);
      const s16x4 lo = ds_read_tr(Vs, vtile_off<D>(key, d >> 3) + (d & 7) * 2);
      const s16x4 hi = ds_read_tr(Vs, vtile_off<D>(key + 8, d >> 3) + (d & 7) * 2);
      const u32x2 lw = __builtin_bit_cast(u32x2, lo), hw = __builtin_bit_cast(u32x2, hi);
      vf[2 * db + u] = __builtin_bit_cast(bf16x8, u32x4{lw[0], lw[1], hw[0], hw[1]});
    }
  }
}

// Both bf16 values of a word at once, by arithmetic in 16-bit halves whose top
// bits catch the carry (one comparison per value would cost a lane mask each).
// 0x8000 in the halves that are not zero / infinite or NaN / NaN:
__device__ __forceinline__ uint32_t halves_set(uint32_t w) {
  return (((w & 0x7fff7fffu) + 0x7fff7fffu) | w) & 0x80008000u;
}
__device__ __forceinline__ uint32_t halves_odd(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t halves_nan(uint32_t w) { return ((w & 0x7fff7fffu) + 0x007f007fu) & 0x80008000u; }

// Whether some value of the fragments is infinite or NaN (exponent all ones).
template <int D>
__device__ __forceinline__ bool odd_values(const bf16x8* vf) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const u32x4 w = __builtin_bit_cast(u32x4, vf[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= halves_odd(w[e]);
  }
  return __ballot(any != 0) != 0;
}

// For a product O^T += V^T P^T in which a row may not see a key whose value is
// infinite or NaN: 0 times that value is NaN, so the fragments are left with
// finite values only, and products of ones count, for each row and column, the
// seen keys that hold +inf, -inf or NaN, and add those: the keys up to `room` of
// groups of 8 not in `bad`, as mask_scores has them, whose weight may have
// underflowed to 0.
template <int D>
__device__ __forceinline__ void take_odd_values(bf16x8* vf, int room, uint32_t bad, f32x16* acc) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
    const float add = kind == 0 ? __builtin_inff() : kind == 1 ? kNegInf : __builtin_nanf("");
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      f32x16 cnt;
#pragma unroll
      for (int r = 0; r < 16; ++r) cnt[r] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 v = __builtin_bit_cast(u32x4, vf[2 * db + u]), x, y;
        int last = room - 4 * g;
        // opaque: nothing of this is worked out for all blocks before the loop,
        // which would cost the attention loop its registers
        asm volatile("" : "+v"(v), "+v"(last));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t inf = halves_set(v[e] ^ (kind == 0 ? 0x7f807f80u : 0xff80ff80u)) ^ 0x80008000u;
          x[e] = ((kind < 2 ? inf : halves_nan(v[e])) >> 15) * 0x3f80u;  // 1.0
          const int r = 8 * u + 2 * e;  // the scores' registers of this word: two keys of one group
          const uint32_t ones = (acc_row(r, 0) <= last ? 0x3f80u : 0u) | (acc_row(r + 1, 0) <= last ? 0x3f800000u : 0u);
          y[e] = (bad >> (r >> 2)) & 1 ? 0u : ones;
        }
        cnt = mfma32x32x16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), cnt);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] += cnt[r] > 0.f ? add : 0.f;
      __builtin_amdgcn_sched_barrier(0);  // one block's counts at a time: this path must not cost the others registers
    }
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    u32x4 v = __builtin_bit_cast(u32x4, vf[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] &= ~((halves_odd(v[e]) >> 15) * 0xffffu);
    vf[i] = __builtin_bit_cast(bf16x8, v);
  }
}

// -inf for the scores of the keys from `first` + `room` + 1 on, and of the groups
// of 8 from `first` on whose bit in `bad` is set.  One comparison a score: the
// row's limit and the keys' end come as one number.
__device__ __forceinline__ void mask_scores(f32x16& s, int room, uint32_t bad) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = acc_row(r, 0) <= room - 4 * g ? s[r] : kNegInf;
  if (bad) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = (bad >> (r >> 2)) & 1 ? kNegInf : s[r];
  }
}

// Host side of each kernel.
constexpr int kFewRows = 32, kTileRows = 128;
constexpr int kMaxSplits = 64;  // key ranges of a tile: one per lane of the wave that combines them
int32_t paged_few_launch(const PagedArgs& a, int D, bool wide, int64_t tiles, hipStream_t s);  // tiles of kFewRows
int32_t paged_tile_launch(const PagedArgs& a, int D, int64_t tiles, hipStream_t s);   // tiles of kTileRows
int32_t paged_finish_launch(const PagedArgs& a, int D, bool few, hipStream_t s);  // split keys; and weights of scores
int32_t paged_score_weights_launch(const PagedArgs& a, hipStream_t s);
int paged_weight_parts(int64_t B, int64_t Hkv, int64_t cap, int64_t N, int64_t G);
int32_t paged_weights_launch(const PagedArgs& a, int D, int parts, float* part, hipStream_t s);

}  // namespace catopt
