// Attention of many tokens a sequence, head_dim padded to 256.
#include "paged_tokens.hpp"

namespace kvssd {

template <>
int launch_paged_tokens_dims<256>(const PagedTokensParams& p, int waves, bool precise, bool, unsigned groups, hipStream_t stream) {
  return precise ? launch_paged_tokens_kernel<256, 4, true, false>(p, groups, stream)
                 : launch_paged_tokens_kernel<256, 4, false, false>(p, groups, stream);
}

}  // namespace kvssd
