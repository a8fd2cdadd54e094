// Attention of many rows a key head over the keys behind a shared prefix (fa_paged_chunk_kernel.h): pages in 16 bits.
#include "fa_paged_chunk_launch.h"

namespace fa {

hipError_t launch_paged_chunk_own(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_chunk_of<false, kOwn>(p, dtype, head_dim, stream);
}

}  // namespace fa
