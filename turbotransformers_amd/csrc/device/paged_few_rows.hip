// The kernels of paged_few_rows.h for rows that see a window or all keys, and sequences on their own.
#include "paged_few_rows.h"

namespace ttmi {

int launch_few_rows(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  TTMI_DISPATCH_FLOAT(dtype, T, { (start_few_rows<T, kWindow>(a, head_dim, stream)); });
  return launch_status("paged_attention");
}

}  // namespace ttmi
