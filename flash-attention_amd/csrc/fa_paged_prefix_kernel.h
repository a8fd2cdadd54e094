// Attention of sequences that share a prefix, a few rows a key head: one launch has two kinds of workgroups.  The first ones attend with a group's rows to the keys that the
// group shares (fa_paged_chunk_kernel.h, kShared), the others have the line of the sequences' own keys (fa_paged_decode_kernel.h); all leave partial results, which a second
// kernel joins.  The first are bound by products and the exponentials, the others by memory: side by side on a compute unit they take little more than the longer of the two.
// 32 sequences of 8 x 4 heads, d = 128, 100 .. 1024 keys of their own behind 8192: 26 to 28 us and 6.4 for the join, 20 for the bytes; 64 of 450 .. 1500 behind 16384 in 8 bits
// 56 to 57 and 7, 31.
#pragma once

#include "fa_paged_chunk_kernel.h"
#include "fa_paged_decode_kernel.h"

namespace fa {

// Keys of a tile of the prefix: the LDS that the others' tiles take holds 64 at d = 128, too.
constexpr int kPrefixKeys = 64;
// Waves a SIMD that registers are to allow.
constexpr int prefix_bound(int head_dim) { return head_dim == 128 ? 2 : 3; }

template <typename T, int D, bool kLse, bool k8>
__global__ void __launch_bounds__(256, prefix_bound(D)) fa_paged_prefix_kernel(const PagedFwdParams p) {
  constexpr int NW = kDecodeBeside(D, k8);
  constexpr int kDecodeLds = DecodeCfg<D, NW, k8>::kLds, kChunkLds = ChunkCfg<D, kPrefixKeys>::kLds;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[kDecodeLds > kChunkLds ? kDecodeLds : kChunkLds];
  const int items = (p.c.HK * p.pre_tiles + 7) / 8 * 8;
  // (the prefix's first: each of them takes longer.  Both kinds in turn: 61 to 62 us where this takes 61.5, 64 sequences behind 16384 keys)
  const int shared = items * p.pre_splits, id = blockIdx.x;
  if (id < shared) {
    paged_chunk<T, D, kLse, k8, true, kPrefixKeys>(p, id % items, id / items, lds_raw);
  } else {
    if (NW < 4 && threadIdx.x >= 64 * NW) return;
    paged_decode<T, D, NW, k8, true, true>(p, id - shared, lds_raw);
  }
}
template <typename T, int D, bool k8>
__global__ void __launch_bounds__(256) paged_prefix_join_kernel(const PagedFwdParams p) {
  paged_decode_join<T, D, k8, true>(p);
}

template <bool k8>
hipError_t launch_prefix_of(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    using T = typename decltype(t)::type;
    const unsigned items = (unsigned)((p.c.HK * p.pre_tiles + 7) / 8 * 8);
    hipLaunchKernelGGL((p.lse ? fa_paged_prefix_kernel<T, d, true, k8> : fa_paged_prefix_kernel<T, d, false, k8>), dim3(items * (unsigned)p.pre_splits + (unsigned)p.groups),
                       dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_decode_join(paged_prefix_join_kernel<T, d, k8>, p, stream);
  });
}

}  // namespace fa
