// Kernels and launches of fa_paged_chunk_kernel.h for pages in 8 bits, for keys behind a shared prefix, and for the prefix.
#pragma once

#include "fa_paged_chunk_kernel.h"

namespace fa {

// Waves a SIMD: as for pages in 16 bits.
template <int D>
constexpr int chunk_waves(bool lse, bool k8) {
  return ChunkCfg<D>::kWaves - (lse || k8 ? 1 : 0);
}

template <typename T, int D, bool kLse, bool k8, int kMode>
__global__ void __launch_bounds__(256, chunk_waves<D>(kLse, k8)) fa_paged_chunk_of_kernel(const PagedFwdParams p) {
  paged_chunk<T, D, kLse, k8, kMode>(p);
}
template <typename T, int D, bool kPrefix>
__global__ void __launch_bounds__(256) paged_chunk_join_of_kernel(const PagedFwdParams p, int lanes) {
  paged_chunk_join<T, D, kPrefix>(p, lanes);
}

template <typename T, int D, bool k8, int kMode>
hipError_t launch_chunk_d(const PagedFwdParams& p, hipStream_t stream) {
  if constexpr (kMode == kShared) {
    const int64_t items = (int64_t)p.c.HK * p.pre_tiles;
    const dim3 grid((unsigned)((items + 7) / 8 * 8), (unsigned)p.pre_splits);
    if (p.lse) hipLaunchKernelGGL((fa_paged_chunk_of_kernel<T, D, true, k8, kShared>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((fa_paged_chunk_of_kernel<T, D, false, k8, kShared>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
  } else {
    const int64_t pairs = (int64_t)p.c.B * p.c.HK, items = pairs * p.nq_tiles;
    const dim3 grid((unsigned)(p.deal ? (pairs + 7) / 8 * 8 * p.nq_tiles : (items + 7) / 8 * 8), (unsigned)p.n_splits);
    if (p.lse || kMode == kOwn) hipLaunchKernelGGL((fa_paged_chunk_of_kernel<T, D, true, k8, kMode>), grid, dim3(256), 0, stream, p);
    else if constexpr (kMode == kAll) hipLaunchKernelGGL((fa_paged_chunk_of_kernel<T, D, false, k8, kAll>), grid, dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (kMode == kAll && p.n_splits <= 1)) return e;
    const int lanes = join_lanes<D>(kMode == kOwn && p.pre_splits > p.n_splits ? p.pre_splits : p.n_splits);
    const int64_t n = items * kChunkRows * kJoinCols<D> * lanes;
    hipLaunchKernelGGL((paged_chunk_join_of_kernel<T, D, kMode == kOwn>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, lanes);
    return hipGetLastError();
  }
}
template <bool k8, int kMode, typename T>
hipError_t launch_chunk_t(const PagedFwdParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_chunk_d<T, 16, k8, kMode>(p, stream);
    case 32: return launch_chunk_d<T, 32, k8, kMode>(p, stream);
    case 64: return launch_chunk_d<T, 64, k8, kMode>(p, stream);
    case 128: return launch_chunk_d<T, 128, k8, kMode>(p, stream);
    default: return hipErrorInvalidValue;
  }
}
template <bool k8, int kMode>
hipError_t launch_chunk_of(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_chunk_t<k8, kMode, _Float16>(p, head_dim, stream) : launch_chunk_t<k8, kMode, __bf16>(p, head_dim, stream);
}

}  // namespace fa
