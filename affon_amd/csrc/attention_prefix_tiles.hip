// Launches of the kernels for prefixes that many rows share.
#include "attention_prefix_tiles.h"

namespace affon {
namespace attention {

void launch_prefix_tiles(const Args& a, int waves, dim3 grid, hipStream_t stream) {
  if (a.p.cache.head_dim == 128) {
    if (waves == 8)
      hipLaunchKernelGGL((prefix_kernel<PrefixKernel<4, 8, 6>>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((prefix_kernel<PrefixKernel<4, 4, 4>>), grid, dim3(256), 0, stream, a);
  } else {
    if (waves == 8)
      hipLaunchKernelGGL((prefix_kernel<PrefixKernel<2, 8, 6>>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((prefix_kernel<PrefixKernel<2, 4, 8>>), grid, dim3(256), 0, stream, a);
  }
}

}  // namespace attention
}  // namespace affon
