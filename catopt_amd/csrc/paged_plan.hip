// A step's tables, slots and positions from its requests' lengths, and the pages
// of finished requests back to the free ones.
//
// Both are latency: what they move is kilobytes.  The new tokens' starts are a
// prefix sum over the sequences, the new pages' places in the pool another one.
// Every workgroup forms the sums it needs by itself, 512 sequences at a time, so
// one launch does without a barrier over workgroups; block 0 writes what belongs
// to the sequences, the others a slice of the tokens each, with the table's new
// entries: a new page's first key is a new token's.  A slice looks its sequences up
// in LDS and takes new pages from the pool by their number, so that no block reads
// what another one writes.
//
// Measured: a step of 8 requests 3.5 us, of 73483 tokens of 500 requests 5.4 (1.4 MB);
// the pages of 16 sequences given back in 2.7, of 512 with half of them ended, of up
// to 16000 keys, in 4.5 + 5.9.  An empty launch takes some 2.
#include "paged.hpp"

namespace catopt {
namespace {

// Threads of a workgroup, sequences at a time, tokens of a slice.  73483 tokens of 500
// requests with 512 threads, captured: 5.2 us in slices of 256, 4.8 of 512, 6.0 of 1024; with 256
// threads (two rounds of sequences) 6.4, with 1024 5.5.
constexpr int NT = 512;

struct ExtendArgs {
  int32_t* table;
  int64_t table_ld;
  const int32_t *lens, *fresh, *pool, *count, *offsets;
  int32_t *starts, *lens_out, *count_out;
  int64_t *positions, *slots;
  FastDiv page;
  int B, N, pool_size, reach;
};

// Inclusive prefix sum over the workgroup, of non-negative values that stay below
// `most` <= 2^30 (they saturate there); `last` receives the whole sum.
__device__ __forceinline__ int block_scan(int v, int most, int* waves, int& last) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v = min(v + u, most);
  }
  __syncthreads();  // the sums before have been read
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  int before = 0;
  last = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) before = last;
    last = min(last + waves[w], most);
  }
  return min(before + v, most);
}

// The largest i of [0, n) with at[i] <= x, where at[0] <= x.
__device__ __forceinline__ int find_last(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Free page j of the step: the pool's last one first, -1 where there is none.
__device__ __forceinline__ int pool_page(const ExtendArgs& a, int count, int j) {
  return j < count ? a.pool[count - 1 - j] : -1;
}

// Of 512 sequences: the first token, the first new page (among the step's), the
// keys before, the pages that hold them.
struct Chunk {
  int start[NT], first[NT], len[NT], held[NT];
};

// `state`: block 0 is the one that writes what belongs to the sequences.
__global__ __launch_bounds__(NT) void paged_extend_kernel(ExtendArgs a, int state) {
  __shared__ Chunk c;
  __shared__ int waves[NT / 64];
  const int tid = threadIdx.x, block = (int)blockIdx.x - state;
  const bool writes_state = block < 0;
  const int t0 = writes_state ? 0 : block * NT, t1 = writes_state ? 0 : min(t0 + NT, a.N);
  const int count = min(max(*a.count, 0), a.pool_size);
  int sum = 0, pages = 0;  // tokens and new pages of the sequences before
  for (int b0 = 0; b0 < a.B; b0 += NT) {
    const int b = b0 + tid, here = min(a.B - b0, NT);
    const int fresh = b < a.B ? min(max(a.fresh[b], 0), a.N) : 0;
    const int len = b < a.B ? min(max(a.lens[b], 0), a.reach) : 0;
    int all, all_pages;
    const int end = min(sum + block_scan(fresh, a.N, waves, all), a.N);
    // what the rows leave of this sequence's tokens: its start is the end before
    const int before = __shfl_up(end, 1, 64);
    if ((tid & 63) == 63) c.start[tid >> 6] = end;
    __syncthreads();
    const int start = tid == 0 ? sum : (tid & 63) ? before : c.start[(tid >> 6) - 1];
    const int after = min(len + (end - start), a.reach);
    const int held = (int)a.page.div(len + a.page.d - 1), need = (int)a.page.div(after + a.page.d - 1) - held;
    const int upto = block_scan(need, 1 << 30, waves, all_pages);
    c.start[tid] = start, c.first[tid] = pages + upto - need, c.len[tid] = len, c.held[tid] = held;
    __syncthreads();
    if (writes_state) {
      if (b < a.B) {
        a.starts[b] = start;
        if (b == a.B - 1) a.starts[a.B] = end;
        a.lens_out[b] = after;
      }
    }
    const int next = min(sum + all, a.N);
    for (int t = max(t0, sum) + tid; t < min(t1, next); t += NT) {
      const int i = find_last(c.start, here, t), key = c.len[i] + t - c.start[i];
      int64_t slot = -1;
      if (key < a.reach) {
        const int p = (int)a.page.div(key);
        const int in = key - p * (int)a.page.d;
        int32_t* entry = a.table + (int64_t)(b0 + i) * a.table_ld + p;
        int id;
        if (p < c.held[i]) {
          id = *entry;
        } else {  // a new page: its first key is a new one, whose token writes the table
          id = pool_page(a, count, c.first[i] + p - c.held[i]);
          if (in == 0) *entry = id;
        }
        if (id >= 0) slot = (int64_t)id * a.page.d + in;
      }
      a.slots[t] = slot;
      a.positions[t] = (int64_t)key + (a.offsets ? a.offsets[b0 + i] : 0);
    }
    sum = next;
    pages += all_pages;
    if (!writes_state && sum >= t1) return;
    __syncthreads();  // the chunk has been read
  }
  for (int t = max(t0, sum) + tid; t < t1; t += NT) a.slots[t] = -1, a.positions[t] = 0;
  if (writes_state && tid == 0) {
    if (a.B == 0) a.starts[0] = 0;
    *a.count_out = max(count - pages, 0);
  }
}

struct ReleaseArgs {
  const int32_t* table;
  int64_t table_ld;
  const int32_t *lens, *count;
  const uint8_t* released;
  int32_t *pool, *lens_out, *count_out;
  int32_t* ws;  // the count, then the pages of each sequence
  FastDiv page;
  int B, n_table, pool_size;
};

// The pages of sequence b that go back, by a wave.
__device__ __forceinline__ int release_count(const ReleaseArgs& a, int b, int& held) {
  held = 0;
  if (!a.released[b]) return 0;
  held = (int)min((int64_t)a.page.div(max(a.lens[b], 0)) + (max(a.lens[b], 0) % a.page.d != 0), (int64_t)a.n_table);
  int n = 0;
  for (int i = threadIdx.x & 63; i < held; i += 64) n += a.table[(int64_t)b * a.table_ld + i] >= 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  return n;
}

// They go to the pool from `to` on, in their order.
__device__ __forceinline__ void release_pages(const ReleaseArgs& a, int b, int held, int64_t to) {
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < held; i0 += 64) {
    const int id = i0 + lane < held ? a.table[(int64_t)b * a.table_ld + i0 + lane] : -1;
    const uint64_t some = __ballot(id >= 0);
    const int64_t at = to + __popcll(some & ((1ull << lane) - 1));
    if (id >= 0 && at < a.pool_size) a.pool[at] = id;
    to += __popcll(some);
  }
}

// Waves, and so sequences, of the form of one launch: 16 sequences take 3.1 us in it,
// 17 in two launches 4.5, the least that two take.
constexpr int RW = 16;

// Few sequences: a wave each, one workgroup.
__global__ __launch_bounds__(64 * RW) void paged_release_one(ReleaseArgs a) {
  __shared__ int counts[RW];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int held = 0, len = 0;
  bool out = false;
  if (wave < a.B) {
    const int n = release_count(a, wave, held);
    out = a.released[wave], len = a.lens[wave];
    if (lane == 0) counts[wave] = n;
  }
  const int count = min(max(*a.count, 0), a.pool_size);
  __syncthreads();
  int64_t before = count, all = count;
  for (int w = 0; w < a.B; ++w) {
    if (w < wave) before += counts[w];
    all += counts[w];
  }
  if (wave < a.B) {
    release_pages(a, wave, held, before);
    if (lane == 0) a.lens_out[wave] = out ? 0 : len;
  }
  if (threadIdx.x == 0) *a.count_out = (int)min(all, (int64_t)a.pool_size);
}

constexpr int RT = 256;

__global__ __launch_bounds__(RT) void paged_release_counts(ReleaseArgs a) {
  const int b = blockIdx.x * (RT / 64) + (threadIdx.x >> 6);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws[0] = min(max(*a.count, 0), a.pool_size);
  if (b >= a.B) return;
  int held;
  const int n = release_count(a, b, held);
  if ((threadIdx.x & 63) == 0) a.ws[1 + b] = n;
}

// Each workgroup adds up the counts before its own sequences.
__global__ __launch_bounds__(RT) void paged_release_pages(ReleaseArgs a) {
  __shared__ int64_t sums[RT / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b0 = blockIdx.x * (RT / 64), b = b0 + wave;
  int64_t n = 0;
  for (int i = threadIdx.x; i < b0; i += RT) n += a.ws[1 + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if (lane == 0) sums[wave] = n;
  __syncthreads();
  int64_t before = a.ws[0];
  for (int w = 0; w < RT / 64; ++w) before += sums[w];
  for (int i = b0; i < min(b, a.B); ++i) before += a.ws[1 + i];
  if (b >= a.B) return;
  const bool out = a.released[b];
  const int len = a.lens[b];
  if (out) {
    const int held = (int)min((int64_t)a.page.div(max(len, 0)) + (max(len, 0) % a.page.d != 0), (int64_t)a.n_table);
    release_pages(a, b, held, before);
  }
  if (lane == 0) {
    a.lens_out[b] = out ? 0 : len;
    if (b == a.B - 1) *a.count_out = (int)min(before + a.ws[1 + b], (int64_t)a.pool_size);
  }
}

Layout vec(const void* p, int64_t size, int64_t n) { return Layout{p, 1, {n, 1, 1, 1}, {1, 1, 1, 1}, size}; }
Layout rows2(const void* p, int64_t size, int64_t n, int64_t ld, int64_t m) {
  return Layout{p, 2, {n, m, 1, 1}, {ld, 1, 1, 1}, size};
}
// Whether two of the outputs, or an output and an input, share memory.
bool clash(std::initializer_list<Layout> outs, std::initializer_list<Layout> ins) {
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    for (auto p = outs.begin(); p != o; ++p)
      if (o->overlaps(*p)) return true;
    for (const Layout& i : ins)
      if (o->overlaps(i)) return true;
  }
  return false;
}

constexpr int64_t kMost = 1LL << 30;

}  // namespace
}  // namespace catopt

using namespace catopt;

extern "C" int32_t catopt_hip_paged_extend(int64_t B, int64_t N, int64_t page_size, int32_t* block_table, int64_t table_ld,
                                           int64_t n_table, const int32_t* kv_lens, const int32_t* new_lens,
                                           const int32_t* free_pages, int64_t n_free, const int32_t* free_count,
                                           const int32_t* offsets, int32_t* q_starts, int64_t* positions, int64_t* slots,
                                           int32_t* kv_lens_out, int32_t* free_count_out, void* stream) {
  if (B < 0 || N < 0 || page_size < 1 || n_table < 0 || table_ld < 0 || n_free < 0) return CATOPT_E_INVAL;
  if (B > (1 << 20) || N >= kMost || n_free >= kMost || page_size >= kMost || n_table >= kMost || n_table * page_size >= kMost)
    return CATOPT_E_UNSUPPORTED;
  if (!q_starts || !free_count || !free_count_out || (N > 0 && (!positions || !slots)) || (n_free > 0 && !free_pages))
    return CATOPT_E_INVAL;
  if (B > 0 && (!kv_lens || !new_lens || !kv_lens_out || (n_table > 0 && !block_table))) return CATOPT_E_INVAL;
  const Layout table = rows2(block_table, 4, B, table_ld, n_table), lens = vec(kv_lens, 4, B), count = vec(free_count, 4, 1);
  const Layout lens_out = vec(kv_lens_out, 4, B), count_out = vec(free_count_out, 4, 1);
  if (table.folded()) return CATOPT_E_INVAL;
  if (clash({table, vec(q_starts, 4, B + 1), vec(positions, 8, N), vec(slots, 8, N), lens_out, count_out},
            {vec(new_lens, 4, B), vec(free_pages, 4, n_free), vec(offsets, 4, B)}))
    return CATOPT_E_INVAL;
  if (clash({table, vec(q_starts, 4, B + 1), vec(positions, 8, N), vec(slots, 8, N)}, {lens, count})) return CATOPT_E_INVAL;
  // lengths and count may be updated in place, and in no other way share memory with an input
  const bool in_place = lens_out.overlaps(lens) || count_out.overlaps(count);
  if (lens_out.overlaps(count) || count_out.overlaps(lens)) return CATOPT_E_INVAL;
  if (lens_out.overlaps(lens) && kv_lens != kv_lens_out) return CATOPT_E_INVAL;
  if (count_out.overlaps(count) && free_count != free_count_out) return CATOPT_E_INVAL;
  ExtendArgs a{};
  a.table = block_table, a.table_ld = table_ld, a.lens = kv_lens, a.fresh = new_lens, a.pool = free_pages;
  a.count = free_count, a.offsets = offsets, a.starts = q_starts, a.lens_out = kv_lens_out, a.count_out = free_count_out;
  a.positions = positions, a.slots = slots, a.page = FastDiv::of(page_size);
  a.B = (int)B, a.N = (int)N, a.pool_size = (int)n_free, a.reach = (int)(n_table * page_size);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t slices = (uint32_t)((N + NT - 1) / NT);
  // in place the tokens go first: their blocks read the lengths that the other one writes
  if (in_place && slices > 0) {
    paged_extend_kernel<<<dim3(slices), dim3(NT), 0, s>>>(a, 0);
    CATOPT_LAUNCH_CHECK();
  }
  paged_extend_kernel<<<dim3(in_place ? 1 : slices + 1), dim3(NT), 0, s>>>(a, 1);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

extern "C" int64_t catopt_hip_paged_release_workspace_bytes(int64_t B) {
  if (B < 0 || B > (1 << 20)) return -1;
  return B > RW ? 4 * (B + 1) : 0;
}

extern "C" int32_t catopt_hip_paged_release(int64_t B, int64_t page_size, const int32_t* block_table, int64_t table_ld,
                                            int64_t n_table, const int32_t* kv_lens, const uint8_t* released,
                                            int32_t* free_pages, int64_t n_free, const int32_t* free_count,
                                            int32_t* kv_lens_out, int32_t* free_count_out, void* workspace,
                                            int64_t workspace_bytes, void* stream) {
  if (B < 0 || page_size < 1 || n_table < 0 || table_ld < 0 || n_free < 0) return CATOPT_E_INVAL;
  const int64_t need = catopt_hip_paged_release_workspace_bytes(B);
  if (need < 0 || n_free >= kMost || page_size >= kMost || n_table >= kMost || n_table * page_size >= kMost)
    return CATOPT_E_UNSUPPORTED;
  if (!free_count || !free_count_out || (n_free > 0 && !free_pages)) return CATOPT_E_INVAL;
  if (B > 0 && (!kv_lens || !released || !kv_lens_out || (n_table > 0 && !block_table))) return CATOPT_E_INVAL;
  const Layout table = rows2(block_table, 4, B, table_ld, n_table), lens = vec(kv_lens, 4, B), count = vec(free_count, 4, 1);
  const Layout lens_out = vec(kv_lens_out, 4, B), count_out = vec(free_count_out, 4, 1), pool = vec(free_pages, 4, n_free);
  if (clash({pool, lens_out, count_out}, {table, vec(released, 1, B)}) || pool.overlaps(lens) || pool.overlaps(count))
    return CATOPT_E_INVAL;
  if (lens_out.overlaps(count) || count_out.overlaps(lens)) return CATOPT_E_INVAL;
  if (lens_out.overlaps(lens) && kv_lens != kv_lens_out) return CATOPT_E_INVAL;
  if (count_out.overlaps(count) && free_count != free_count_out) return CATOPT_E_INVAL;
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4)) return CATOPT_E_WORKSPACE;
  ReleaseArgs a{};
  a.table = block_table, a.table_ld = table_ld, a.lens = kv_lens, a.count = free_count, a.released = released;
  a.pool = free_pages, a.lens_out = kv_lens_out, a.count_out = free_count_out, a.ws = static_cast<int32_t*>(workspace);
  a.page = FastDiv::of(page_size), a.B = (int)B, a.n_table = (int)n_table, a.pool_size = (int)n_free;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (B <= RW) {
    paged_release_one<<<dim3(1), dim3(64 * RW), 0, s>>>(a);
    CATOPT_LAUNCH_CHECK();
    return CATOPT_OK;
  }
  const dim3 grid((uint32_t)((B + RT / 64 - 1) / (RT / 64)));
  paged_release_counts<<<grid, dim3(RT), 0, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  paged_release_pages<<<grid, dim3(RT), 0, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}
