// Launches of the kernels for prefixes that many rows share.
#include "attention_prefix_tiles.h"

namespace affon {
namespace attention {

template <typename K>
void launch_prefix(const Args& a, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL(prefix_kernel<K>, grid, dim3(K::kThreads), 0, stream, a);
}

void launch_prefix_tiles(const Args& a, int waves, dim3 grid, hipStream_t stream) {
  const int D = a.p.cache.head_dim;
  if (a.p.cache.dtype == AFFON_ROCM_BF16) {
    if (D == 128 && waves == 8) launch_prefix<PrefixKernel<4, 8, 6>>(a, grid, stream);
    if (D == 128 && waves == 4) launch_prefix<PrefixKernel<4, 4, 4>>(a, grid, stream);
    if (D == 64 && waves == 8) launch_prefix<PrefixKernel<2, 8, 6>>(a, grid, stream);
    if (D == 64 && waves == 4) launch_prefix<PrefixKernel<2, 4, 8>>(a, grid, stream);
    return;
  }
  switch (D) {
    case 64: return launch_prefix<PrefixF32<64>>(a, grid, stream);
    case 80: return launch_prefix<PrefixF32<80>>(a, grid, stream);
    case 96: return launch_prefix<PrefixF32<96>>(a, grid, stream);
    default: return launch_prefix<PrefixF32<128>>(a, grid, stream);
  }
}

}  // namespace attention
}  // namespace affon
