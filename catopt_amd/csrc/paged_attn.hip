// Paged attention: the choice of kernels and the workspace.
#include "paged_attn.hpp"

namespace catopt {
namespace {

struct Plan {
  bool few, wide;
  int splits, min_keys, parts;
  int64_t tiles, part_floats, stat_floats, score_floats, weight_floats;
  int64_t bytes() const { return 4 * (part_floats + stat_floats + score_floats + weight_floats); }
};

// Key ranges of 128-row tiles by their estimated time, were every sequence as
// long as its table.  A workgroup takes a tile of 64 keys in 1.7 us alone on
// its CU and 2.4 beside another (D = 64: 1 and 1.5), its start and masked tiles
// shared out (1.35 and 2.3 without, which chose worse: 150 tokens each of two
// sequences over 1650 keys 32.6 us for 29.1); more workgroups than 512 are
// priced as rounds (at D = 64, where three fit a CU, 513 to 768 are priced a
// round that they do not run).  Ranges cost a launch, 5.5 us, and their
// numerators' way through memory, at 6 TB/s.  Measured, one range against the
// ranges chosen (us): 64 tokens over 564 keys, 32 heads on 8, 18.0 and 14.2; 33 to
// 171 tokens of five sequences, 12 heads of 64, 40 and 21; a prompt of 512 tokens
// and a table as long 17 and 20 (one chosen), but against a table of 2048 keys or
// more it gets four ranges and takes 21.
int tile_splits(int64_t groups, int64_t rows, int64_t D, int64_t cap) {
  const double alone = D == 128 ? 1.7 : 1.0, beside = D == 128 ? 2.4 : 1.5;
  double best = 0;
  int splits = 1;
  for (int s = 1; s <= kMaxSplits; ++s) {
    const int64_t keys = ((cap + s - 1) / s + 127) / 128 * 128, wgs = groups * s;
    const double rounds = wgs <= 512 ? 1 : wgs / 512.0, tile = wgs <= 256 ? alone : beside;
    const double us = rounds * (keys / 64) * tile + (s > 1 ? 5.5 + (double)rows * s * D * 8 / 6e6 : 0);
    if (s == 1 || us < best) best = us, splits = s;
    if (keys <= 128) break;
  }
  return splits;
}

// The kernel and the key ranges by sizes that the host knows.
//
// Few rows: 32-row tiles whenever the sequences have 32 rows per key head or
// fewer on average.
//
// One range, and so one launch, where the table reaches 1024 keys or fewer and
// the CUs hold every tile at once: the wide kernel then takes 12 us at 1000
// keys, 32 query heads on 8, and 10.7 (the host's time) at 500, where split
// keys and their combination take 14.9.
//
// Ranges: few-row calls read K and V at the rate of HBM, so their ranges only
// have to fill the CUs and even out the sequences: at most 64 to a tile and
// 16384 workgroups in all (those behind a sequence's keys end at once).  A range
// is 256 keys at least; 128 where the table's reach is less than 256 for each
// of the 512 workgroups that the CUs hold; 1024 where it is 4096 for each (a
// step of 32 sequences of 300 to 16000 keys: 100.6 us, 106.6 with 256; at eight
// sequences of 2000 to 12000 they are level).
//
// 128-row tiles: see tile_splits.
//
// All of this goes by the tables' reach and the average of the rows, so it is at
// its best where tables are about as wide as the longest sequence and no entry is
// idle.  Eight steps of 2000 keys take 17 us, against tables of 32768 keys 33; of
// 500 keys 10 and 21.  A chunk of 2048 tokens takes 56 us alone and 195 beside 255
// idle entries, which put it on 32-row tiles.  32 steps of 16000 keys and a chunk
// of 512 tokens over 4096 keys take 394 us in one call, 330 and 55 in two.
Plan plan_of(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d, int64_t cap, bool weights) {
  Plan p{};
  const int64_t G = Hq / Hkv, D = d <= 64 ? 64 : 128;
  p.few = N * G <= kFewRows * B;
  p.tiles = paged_tiles(N, G, B, p.few ? kFewRows : kTileRows);
  const int64_t groups = p.tiles * Hkv;
  const int64_t rows = N * Hq;
  if (p.few) {
    int64_t s = 16384 / groups;
    const int64_t per_slot = groups * cap / 512;
    p.min_keys = per_slot >= 4096 ? 1024 : per_slot >= 256 ? 256 : 128;
    p.wide = groups <= 256 && cap <= 1024;
    const int64_t most = p.wide ? 1 : (cap + p.min_keys - 1) / p.min_keys;
    if (s > kMaxSplits) s = kMaxSplits;
    if (s > most) s = most;
    p.splits = s < 1 ? 1 : (int)s;
  } else {
    p.min_keys = 128;
    p.splits = tile_splits(groups, rows, D, cap);
  }
  p.part_floats = p.splits > 1 ? ((2 * rows * p.splits + 3) & ~(int64_t)3) + rows * p.splits * D : 0;
  if (weights) {
    p.stat_floats = (rows + 3) & ~(int64_t)3;
    if (p.few && rows * cap <= (1LL << 28)) {
      p.score_floats = rows * cap;
    } else {
      p.parts = paged_weight_parts(B, Hkv, cap, N, G);
      p.weight_floats = p.parts > 1 ? p.parts * B * Hkv * cap : 0;
    }
  }
  return p;
}

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int64_t catopt_hip_paged_attn_workspace_bytes(int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d,
                                                         int64_t n_table, int64_t page_size, int32_t weights) {
  const int64_t lim = 1LL << 30;
  if (B < 0 || N < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || d < 8 || d > 128 || d % 8) return -1;
  if (n_table < 0 || page_size < 8 || page_size % 8) return -1;
  if (B > (1 << 20) || N >= lim || Hq > 65535 || N * Hq >= lim || B * Hkv >= lim) return -1;
  if (n_table > lim || page_size > lim || n_table * page_size >= lim) return -1;
  if (B == 0 || N == 0) return 0;
  return plan_of(B, N, Hq, Hkv, d, n_table * page_size, weights != 0).bytes();
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
  if (!(scale > 0.f) || !__builtin_isfinite(scale * kLog2e)) return CATOPT_E_UNSUPPORTED;
  const int64_t need = catopt_hip_paged_attn_workspace_bytes(B, N, Hq, Hkv, d, n_table, page_size, weights_out != nullptr);
  if (need < 0) return CATOPT_E_UNSUPPORTED;
  if (B == 0 || (N == 0 && !weights_out)) return CATOPT_OK;
  if ((N > 0 && (!q || !o)) || !kv_lens || !q_starts || !strides || (n_table > 0 && !block_table)) return CATOPT_E_INVAL;
  if (n_pages > 0 && (!k_pages || !v_pages)) return CATOPT_E_INVAL;
  const Strides rows(strides, {N, Hq, n_pages, Hkv, page_size, n_pages, Hkv, page_size, N, Hq}, 8);
  const Strides sums(strides + 10, {B, Hkv, B, Hkv}, 1);
  if (!rows.fit || !sums.fit) return CATOPT_E_INVAL;
  const int64_t *s = rows.s, *w = sums.s;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o)) return CATOPT_E_INVAL;
  if (weights_in && !weights_out) return CATOPT_E_INVAL;
  const Layout out = layout3(o, 2, N, s[8], Hq, s[9], d), lq = layout3(q, 2, N, s[0], Hq, s[1], d);
  const Layout lk = layout_pages(k_pages, 2, n_pages, Hkv, page_size, d, s + 2);
  const Layout lv = layout_pages(v_pages, 2, n_pages, Hkv, page_size, d, s + 5);
  if (out.folded() || out.overlaps(lq) || out.overlaps(lk) || out.overlaps(lv)) return CATOPT_E_INVAL;
  if (weights_out) {
    const int64_t cap = n_table * page_size;
    const Layout wo = layout3(weights_out, 4, B, w[2], Hkv, w[3], cap);
    const Layout wi = layout3(weights_in, 4, B, w[0], Hkv, w[1], cap);
    if (wo.folded() || wo.overlaps(lq) || wo.overlaps(lk) || wo.overlaps(lv) || wo.overlaps(out)) return CATOPT_E_INVAL;
    if (weights_in && ((wo.overlaps(wi) && !wo.same(wi)) || out.overlaps(wi))) return CATOPT_E_INVAL;
  }
  // the rows of one load lie within 31 bits of its resource's base
  if (s[4] > (1 << 26) || s[7] > (1 << 26)) return CATOPT_E_UNSUPPORTED;
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return CATOPT_E_WORKSPACE;
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k_pages);
  a.v = static_cast<const uint16_t*>(v_pages), a.o = static_cast<uint16_t*>(o);
  a.q_t = s[0], a.q_h = s[1], a.k_p = s[2], a.k_h = s[3], a.k_s = s[4], a.v_p = s[5], a.v_h = s[6], a.v_s = s[7];
  a.o_t = s[8], a.o_h = s[9], a.wi_b = w[0], a.wi_h = w[1], a.wo_b = w[2], a.wo_h = w[3];
  a.table = block_table, a.lens = kv_lens, a.starts = q_starts, a.table_ld = table_ld, a.n_pages = n_pages, a.N = N;
  a.m_out = m_out, a.l_out = l_out, a.w_in = weights_in, a.w_out = weights_out;
  a.page = FastDiv::of(page_size), a.group = FastDiv::of(Hq / Hkv);
  a.q_heads = FastDiv::of(Hq), a.k_heads = FastDiv::of(Hkv);
  a.B = (int)B, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv), a.d = (int)d, a.cap = (int)(n_table * page_size);
  a.normalize = normalize, a.causal = causal != 0, a.scale = scale;
  const Plan p = N == 0 ? Plan{} : plan_of(B, N, Hq, Hkv, d, a.cap, weights_out != nullptr);
  float* ws = static_cast<float*>(workspace);
  a.splits = p.splits, a.min_keys = p.min_keys, a.ranges = FastDiv::of(p.splits < 1 ? 1 : p.splits);
  a.part = ws;
  ws += p.part_floats;
  if (weights_out) {
    a.row_log = ws;
    ws += p.stat_floats;
    a.scores = p.score_floats ? ws : nullptr;
    ws += p.score_floats;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int D = d <= 64 ? 64 : 128;
  if (N == 0) return paged_weights_launch(a, D, 1, nullptr, st);  // no new tokens: the sums so far
  int32_t r = p.few ? paged_few_launch(a, D, p.wide, p.tiles, st) : paged_tile_launch(a, D, p.tiles, st);
  if (r == CATOPT_OK && p.splits > 1) r = paged_finish_launch(a, D, p.few, st);
  if (r == CATOPT_OK && weights_out && !(a.scores && p.splits > 1)) r = paged_weights_launch(a, D, p.parts, ws, st);
  return r;
}
