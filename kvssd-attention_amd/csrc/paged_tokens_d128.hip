// Attention of many tokens a sequence, head_dim padded to 128.
#include "paged_tokens.hpp"

namespace kvssd {

template <>
int launch_paged_tokens_dims<128>(const PagedTokensParams& p, int waves, bool precise, bool own, unsigned groups, hipStream_t stream) {
  if (own) return launch_paged_tokens_kernel<128, 4, false, true>(p, groups, stream);
  if (waves == 8) return launch_paged_tokens_kernel<128, 8, false, false>(p, groups, stream);
  return precise ? launch_paged_tokens_kernel<128, 4, true, false>(p, groups, stream)
                 : launch_paged_tokens_kernel<128, 4, false, false>(p, groups, stream);
}

}  // namespace kvssd
