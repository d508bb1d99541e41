// The kernels of paged_sight.h in bf16.
#include "paged_sight.h"

namespace ttmi {
void launch_sight_bf16(const SightLaunch& l, int64_t head_dim, hipStream_t stream) { start_sight<bf16>(l, head_dim, stream); }
}  // namespace ttmi
