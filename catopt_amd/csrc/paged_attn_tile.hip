// The 128-row kernel of paged attention (see the header for how it works).
#include "paged_attn_tile.hpp"

namespace catopt {
namespace {

template <int D>
__global__ __launch_bounds__((kTileThreads), (D == 64 ? 3 : 2)) void paged_tile_kernel(PagedArgs a, int tiles) {
  paged_tile_rows<D, kRows>(a, a, blockIdx.x, tiles);
}

template <int D>
int32_t launch(const PagedArgs& a, int64_t tiles, hipStream_t s) {
  static bool done[kDevices] = {};
  const int32_t r = allow_lds(reinterpret_cast<const void*>(&paged_tile_kernel<D>), TileLds<D>::BYTES, done);
  if (r != CATOPT_OK) return r;
  const int64_t blocks = tiles * a.splits * a.Hkv;
  if (!grid_fits(blocks, kTileThreads)) return CATOPT_E_UNSUPPORTED;
  paged_tile_kernel<D><<<dim3((uint32_t)blocks), dim3(kTileThreads), TileLds<D>::BYTES, s>>>(a, (int)tiles);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_tile_launch(const PagedArgs& a, int D, int64_t tiles, hipStream_t s) {
  return D == 128 ? launch<128>(a, tiles, s) : launch<64>(a, tiles, s);
}

}  // namespace catopt
