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
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_chunk_join_8bit_kernel(const PagedFwdParams p, int lanes) {
  paged_chunk_join<T, D>(p, lanes);
}

template <typename T, int D>
hipError_t launch_d(const PagedFwdParams& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.c.B * p.c.HK * p.nq_tiles;
  const int64_t pairs = (int64_t)p.c.B * p.c.HK;
  const dim3 grid((unsigned)(p.deal ? (pairs + 7) / 8 * 8 * p.nq_tiles : (items + 7) / 8 * 8), (unsigned)p.n_splits);
  if (p.lse) hipLaunchKernelGGL((fa_paged_chunk_8bit_kernel<T, D, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((fa_paged_chunk_8bit_kernel<T, D, false>), grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_splits <= 1) return e;
  const int lanes = join_lanes<D>(p.n_splits);
  const int64_t n = items * kChunkRows * kJoinCols<D> * lanes;
  hipLaunchKernelGGL((paged_chunk_join_8bit_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, lanes);
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

hipError_t launch_paged_chunk_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
