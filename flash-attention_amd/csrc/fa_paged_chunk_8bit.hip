// Attention of many rows a key head over pages in 8 bits (fa_paged_chunk_kernel.h).
#include "fa_paged_chunk_launch.h"

namespace fa {

hipError_t launch_paged_chunk_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_chunk_of<true, kAll>(p, dtype, head_dim, stream);
}

}  // namespace fa
