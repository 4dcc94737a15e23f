// INT4 instances of the paged decode kernel, head_dim up to 128 (paged_decode.hpp).
#include "paged_decode.hpp"

namespace kvssd {
template <>
int launch_paged_dims<4, 128>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream) {
  if (gp == 1) return launch_paged_shape<4, 128, 1>(p, precise, stream);
  if (gp == 2) return launch_paged_shape<4, 128, 2>(p, precise, stream);
  return launch_paged_shape<4, 128, 4>(p, precise, stream);
}
}  // namespace kvssd
