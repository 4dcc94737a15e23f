// Attention of many tokens a sequence, head_dim padded to 128.
#include "paged_tokens.hpp"

namespace kvssd {

template <>
int launch_paged_tokens_dims<128>(const PagedTokensParams& p, int columns, bool precise, unsigned groups, hipStream_t stream) {
  if (columns == 2) return launch_paged_tokens_kernel<128, 2, false>(p, groups, stream);
  return precise ? launch_paged_tokens_kernel<128, 1, true>(p, groups, stream)
                 : launch_paged_tokens_kernel<128, 1, false>(p, groups, stream);
}

}  // namespace kvssd
