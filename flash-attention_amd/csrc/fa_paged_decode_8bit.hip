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

template <typename T, int D>
hipError_t launch_d(const PagedFwdParams& p, hipStream_t stream) {
  const unsigned pairs = (unsigned)(p.c.B * p.c.HK);
  const dim3 grid(p.groups > 0 ? (unsigned)p.groups : pairs);
  if (p.wide == 2) hipLaunchKernelGGL((paged_decode_wide_stream_8bit_kernel<T, D>), grid, dim3(64 * kDecodeWide8), 0, stream, p);
  else if (p.wide) hipLaunchKernelGGL((fa_paged_decode_8bit_kernel<T, D, kDecodeWide8>), grid, dim3(64 * kDecodeWide8), 0, stream, p);
  else hipLaunchKernelGGL((fa_paged_decode_8bit_kernel<T, D, kDecodeWaves8>), grid, dim3(64 * kDecodeWaves8), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.groups == 0) return e;
  const unsigned rows = (unsigned)(p.c.max_sq * p.c.G), side = pairs < 1024 ? 1024 / pairs : 1;  // (workgroups beside each other for a pair's rows)
  hipLaunchKernelGGL((paged_decode_join_8bit_kernel<T, D>), dim3(pairs, rows < side ? rows : side), dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(const PagedFwdParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_d<T, 16>(p, stream);
    case 32: return launch_d<T, 32>(p, stream);
    case 64: return launch_d<T, 64>(p, stream);
    case 128: return launch_d<T, 128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_paged_decode_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
