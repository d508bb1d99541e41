// The kernels of paged_sight.h in f16.
#include "paged_sight.h"

namespace ttmi {
void launch_sight_f16(const SightLaunch& l, int64_t head_dim, hipStream_t stream) { start_sight<f16>(l, head_dim, stream); }
}  // namespace ttmi
