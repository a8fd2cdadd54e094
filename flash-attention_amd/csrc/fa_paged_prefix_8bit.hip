// Attention of groups of sequences over the keys that each group shares (fa_paged_chunk_kernel.h): pages in 8 bits.
#include "fa_paged_chunk_launch.h"

namespace fa {

hipError_t launch_paged_prefix_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_chunk_of<true, kShared>(p, dtype, head_dim, stream);
}

}  // namespace fa
