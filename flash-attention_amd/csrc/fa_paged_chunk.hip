// Attention of a chunk of new tokens over a paged cache: G * Lq rows a key head, any number of them.
//
// The forward kernel's plan (fa_fwd_kernel.h): a workgroup of four waves owns 128 rows, 32 a wave, and streams tiles of K and V through a double
// buffer in LDS; S^T = K Q^T and O^T = V^T P^T keep a row in a lane, its maximum moves only where it has to.  What differs: a tile's rows come from pages, in
// groups of 16 that lie in one page each (their addresses are made by scalar instructions, their pages asked for a step ahead through the scalar cache),
// rows are heads of a group times tokens, so that a key head's keys are read once per 128 of them, and the causal mask is aligned at the end.
// Bound by the matrix cores and the exponentials; launches of few rows and many keys share a row tile's keys among workgroups (n_splits) and
// join their partial results in a second kernel.
#include "fa_paged_chunk_kernel.h"

namespace fa {

template <typename T, int D, bool kLse>
__global__ void __launch_bounds__(256, ChunkCfg<D>::kWaves - (kLse ? 1 : 0)) fa_paged_chunk_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[ChunkCfg<D>::kLds];
  paged_chunk<T, D, kLse, false, false>(p, blockIdx.x, blockIdx.y, lds_raw);
}

namespace {

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const PagedFwdParams p, int lanes) {
  paged_chunk_join<T, D>(p, lanes);
}

}  // namespace

hipError_t launch_paged_chunk_join(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    constexpr int D = d;
    const int lanes = join_lanes<D>(p.n_splits);
    const int64_t n = (int64_t)p.c.B * p.c.HK * p.nq_tiles * kChunkRows * kJoinCols<D> * lanes;
    hipLaunchKernelGGL((paged_chunk_join_kernel<typename decltype(t)::type, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, lanes);
    return hipGetLastError();
  });
}

hipError_t launch_paged_chunk(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    using T = typename decltype(t)::type;
    return launch_chunk(p.lse ? fa_paged_chunk_kernel<T, d, true> : fa_paged_chunk_kernel<T, d, false>, p, dtype, head_dim, stream);
  });
}

}  // namespace fa
