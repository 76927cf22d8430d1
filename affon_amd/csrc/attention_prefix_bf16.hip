// The attention kernels of prefixes that sequences share, over bf16 caches.
#include "attention.h"

namespace affon {
namespace attention {

void launch_prefix_bf16(const Args& a, Shape shape, dim3 grid, hipStream_t stream) { launch_head<BF16, kPrefix>(a, shape, grid, stream); }

}  // namespace attention
}  // namespace affon
