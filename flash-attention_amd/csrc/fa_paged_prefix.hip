// Attention of sequences that share a prefix, a few rows a key head (fa_paged_prefix_kernel.h): pages in 16 bits.
#include "fa_paged_prefix_kernel.h"

namespace fa {

hipError_t launch_paged_prefix(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_prefix_of<false>(p, dtype, head_dim, stream);
}

}  // namespace fa
