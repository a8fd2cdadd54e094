// Attention of a few rows a key head over the keys behind a shared prefix, whose parts it adds (fa_paged_decode_kernel.h): pages in 16 bits.
#include "fa_paged_decode_launch.h"

namespace fa {

hipError_t launch_paged_decode_own(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_decode_of<false, true>(p, dtype, head_dim, stream);
}

}  // namespace fa
