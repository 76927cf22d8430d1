// The attention kernels over bf16 caches.
#include "attention.h"

namespace affon {
namespace attention {

void launch_bf16(const Args& a, Shape shape, dim3 grid, hipStream_t stream) { launch_head<BF16>(a, shape, grid, stream); }

}  // namespace attention
}  // namespace affon
