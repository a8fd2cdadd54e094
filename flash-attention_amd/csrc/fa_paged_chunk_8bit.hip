// Attention of many rows a key head over pages in 8 bits (fa_paged_chunk_kernel.h).
#include "fa_paged_chunk_kernel.h"

namespace fa {

namespace {

// Tiles are larger than over pages in 16 bits, for two waves a SIMD at d = 128 (64 keys, 4 x 1024 tokens over 4096 .. 8192 keys, 8 x 4 heads 424 us, 32 keys 454, three
// waves of these, with registers in scratch, 488; 16 x 1024 over 5120 1414 / 1477) and for fewer meetings at d <= 32 (128 keys, 4 x 1024 tokens over 8192 keys, 8 x 2
// heads of 32 141, 64 keys 169).
template <int D>
constexpr int kKeys8 = D <= 32 ? 128 : 64;
template <typename T, int D, bool kLse>
__global__ void __launch_bounds__(256, 2) fa_paged_chunk_8bit_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[ChunkCfg<D, kKeys8<D>>::kLds];
  paged_chunk<T, D, kLse, true, false, kKeys8<D>>(p, blockIdx.x, blockIdx.y, lds_raw);
}

}  // namespace

hipError_t launch_paged_chunk_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    using T = typename decltype(t)::type;
    return launch_chunk(p.lse ? fa_paged_chunk_8bit_kernel<T, d, true> : fa_paged_chunk_8bit_kernel<T, d, false>, p, dtype, head_dim, stream);
  });
}

}  // namespace fa
