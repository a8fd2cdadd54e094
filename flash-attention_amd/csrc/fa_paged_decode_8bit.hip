// Attention of a few rows a key head over pages in 8 bits (fa_paged_decode_kernel.h).
#include "fa_paged_decode_launch.h"

namespace fa {

hipError_t launch_paged_decode_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_decode_of<true, false>(p, dtype, head_dim, stream);
}

}  // namespace fa
