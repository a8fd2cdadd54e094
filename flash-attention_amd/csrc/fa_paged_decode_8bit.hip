// Attention of a few rows a key head over pages in 8 bits (fa_paged_decode_kernel.h).
#include "fa_paged_decode_kernel.h"

namespace fa {

namespace {

// (as many workgroups as decode_resident of fa_paged_api.hip has on a compute unit; at d = 128 two by LDS, too)
template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, D == 128 ? 2 : D == 64 ? 3 : 4) fa_paged_decode_8bit_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[DecodeCfg<D, NW, true>::kLds];
  paged_decode<T, D, NW, true, false, NW != kDecodeWide8>(p, blockIdx.x, lds_raw);
}
template <typename T, int D>
__global__ void __launch_bounds__(64 * kDecodeWide8, D == 128 ? 2 : D == 64 ? 3 : 4) paged_decode_wide_stream_8bit_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[DecodeCfg<D, kDecodeWide8, true>::kLds];
  paged_decode<T, D, kDecodeWide8, true, false, true>(p, blockIdx.x, lds_raw);
}
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_decode_join_8bit_kernel(const PagedFwdParams p) {
  paged_decode_join<T, D, true, false>(p);
}

}  // namespace

hipError_t launch_paged_decode_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    using T = typename decltype(t)::type;
    constexpr int D = d;
    const auto kernel = p.wide == 2 ? paged_decode_wide_stream_8bit_kernel<T, D>
                                    : p.wide ? fa_paged_decode_8bit_kernel<T, D, kDecodeWide8> : fa_paged_decode_8bit_kernel<T, D, kDecodeWaves8>;
    return launch_decode(kernel, p.wide ? kDecodeWide8 : kDecodeWaves8, paged_decode_join_8bit_kernel<T, D>, p, stream);
  });
}

}  // namespace fa
