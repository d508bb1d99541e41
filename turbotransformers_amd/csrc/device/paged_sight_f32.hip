// The kernels of paged_sight.h in fp32.
#include "paged_sight.h"

namespace ttmi {
void launch_sight_f32(const SightLaunch& l, int64_t head_dim, hipStream_t stream) { start_sight<float>(l, head_dim, stream); }
}  // namespace ttmi
