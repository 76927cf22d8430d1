// The attention kernels of prefixes that sequences share, over f32 caches.
#include "attention.h"

namespace affon {
namespace attention {

void launch_prefix_f32(const Args& a, Shape shape, dim3 grid, hipStream_t stream) { launch_head<F32, kPrefix>(a, shape, grid, stream); }

}  // namespace attention
}  // namespace affon
