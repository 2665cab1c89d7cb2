// The few-row kernel of paged attention (see the header for how it works).
#include "paged_attn_few.hpp"

namespace catopt {
namespace {

template <int D, bool WIDE>
__global__ __launch_bounds__((Few<D, WIDE>::NT), 2) void paged_few_kernel(PagedArgs a) {
  paged_few<D, Few<D, WIDE>, kRows>(a, blockIdx.x);
}

template <int D, bool WIDE>
int32_t launch(const PagedArgs& a, int64_t tiles, hipStream_t s) {
  using L = Few<D, WIDE>;
  static bool done[kDevices] = {};
  const int32_t r = allow_lds(reinterpret_cast<const void*>(&paged_few_kernel<D, WIDE>), L::BYTES, done);
  if (r != CATOPT_OK) return r;
  const int64_t blocks = tiles * a.splits * a.Hkv;
  if (!grid_fits(blocks, L::NT)) return CATOPT_E_UNSUPPORTED;
  paged_few_kernel<D, WIDE><<<dim3((uint32_t)blocks), dim3(L::NT), L::BYTES, s>>>(a);
  CATOPT_LAUNCH_CHECK();
  return CATOPT_OK;
}

}  // namespace

int32_t paged_few_launch(const PagedArgs& a, int D, bool wide, int64_t tiles, hipStream_t s) {
  if (D == 128) return wide ? launch<128, true>(a, tiles, s) : launch<128, false>(a, tiles, s);
  return wide ? launch<64, true>(a, tiles, s) : launch<64, false>(a, tiles, s);
}

}  // namespace catopt
