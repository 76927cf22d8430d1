// The attention kernels over shared prefixes and what follows them, f32 caches.
#include "attention.h"

namespace affon {
namespace attention {

void launch_parts_f32(const Parts& parts, Shape shape, dim3 grid, hipStream_t stream) {
  launch_head<F32, kParts>(parts, shape, grid, stream);
}

}  // namespace attention
}  // namespace affon
