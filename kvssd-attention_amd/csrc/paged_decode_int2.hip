// INT2 instances of the paged decode kernel (paged_decode.hpp).
#include "paged_decode.hpp"

namespace kvssd {
int launch_paged_int2(const PagedDecodeParams& p, int dp, int nt, bool precise, hipStream_t stream) {
  return launch_paged_bits<2>(p, dp, nt, precise, stream);
}
}  // namespace kvssd
