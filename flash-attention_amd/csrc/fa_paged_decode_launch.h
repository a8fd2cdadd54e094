// Kernels and launches of fa_paged_decode_kernel.h for pages in 8 bits and for keys behind a shared prefix.
#pragma once

#include "fa_paged_decode_kernel.h"

namespace fa {

// Waves a SIMD that registers are to allow; LDS allows two (8 bits, d = 128; 16 bits one) or more.
constexpr int decode_bound_of(int head_dim, int waves, bool k8) {
  return k8 ? (head_dim == 128 ? 2 : head_dim == 64 ? 3 : 4) : (head_dim == 128 ? 1 : (waves == 8 ? 2 : (head_dim == 64 ? 3 : 4)));
}

template <typename T, int D, int NW, bool k8, bool kPrefix>
__global__ void __launch_bounds__(64 * NW, decode_bound_of(D, NW, k8)) fa_paged_decode_of_kernel(const PagedFwdParams p) {
  paged_decode<T, D, NW, k8, kPrefix>(p);
}
template <typename T, int D, bool k8, bool kPrefix>
__global__ void __launch_bounds__(256) paged_decode_join_of_kernel(const PagedFwdParams p) {
  paged_decode_join<T, D, k8, kPrefix>(p);
}

template <typename T, int D, bool k8, bool kPrefix>
hipError_t launch_decode_d(const PagedFwdParams& p, hipStream_t stream) {
  constexpr int kWide = k8 ? kDecodeWide8 : kDecodeWide(D), kUsual = k8 ? kDecodeWaves8 : kDecodeWaves(D);
  const unsigned pairs = (unsigned)(p.c.B * p.c.HK);
  const dim3 grid(p.groups > 0 ? (unsigned)p.groups : pairs);
  if (p.wide) hipLaunchKernelGGL((fa_paged_decode_of_kernel<T, D, kWide, k8, kPrefix>), grid, dim3(64 * kWide), 0, stream, p);
  else hipLaunchKernelGGL((fa_paged_decode_of_kernel<T, D, kUsual, k8, kPrefix>), grid, dim3(64 * kUsual), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.groups == 0) return e;
  const unsigned rows = (unsigned)(p.c.max_sq * p.c.G), side = pairs < 1024 ? 1024 / pairs : 1;  // (workgroups beside each other for a pair's rows)
  hipLaunchKernelGGL((paged_decode_join_of_kernel<T, D, k8, kPrefix>), dim3(pairs, rows < side ? rows : side), dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <bool k8, bool kPrefix, typename T>
hipError_t launch_decode_t(const PagedFwdParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_decode_d<T, 16, k8, kPrefix>(p, stream);
    case 32: return launch_decode_d<T, 32, k8, kPrefix>(p, stream);
    case 64: return launch_decode_d<T, 64, k8, kPrefix>(p, stream);
    case 128: return launch_decode_d<T, 128, k8, kPrefix>(p, stream);
    default: return hipErrorInvalidValue;
  }
}
template <bool k8, bool kPrefix>
hipError_t launch_decode_of(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_decode_t<k8, kPrefix, _Float16>(p, head_dim, stream) : launch_decode_t<k8, kPrefix, __bf16>(p, head_dim, stream);
}

}  // namespace fa
