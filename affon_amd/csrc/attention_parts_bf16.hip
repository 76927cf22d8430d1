// The attention kernels over shared prefixes and what follows them, bf16 caches.
#include "attention.h"

namespace affon {
namespace attention {

void launch_parts_bf16(const Parts& parts, Shape shape, dim3 grid, hipStream_t stream) {
  launch_head<BF16, kParts>(parts, shape, grid, stream);
}

}  // namespace attention
}  // namespace affon
