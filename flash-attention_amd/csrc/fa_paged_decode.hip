// Attention of a few rows a key head (decoding: one new token of each sequence, or a handful, times the heads of a group) over a paged cache:
// every key and value is read once and used for at most 32 rows, a stream of K and V that HBM bounds.
//
// A wave owns 32-key tiles: it stages them into a double buffer of its own by direct-to-LDS loads, counts its outstanding loads instead of meeting the
// other waves, and multiplies in the orientation S^T = K Q^T, O^T = V^T P^T (a lane is a row); the workgroup's waves join their partial results in
// LDS at the end of a pair.  Lengths differ and are known on the device only, so the launch does not cut sequences into equal numbers of pieces: all
// units of kDecodeUnit keys of all pairs are laid out in one line, and each of the resident workgroups takes an equal share of it - the end of one
// pair, some whole pairs, the beginning of another.  Pairs that more than one workgroup has touched are joined by a second kernel.  Pairs that fill
// the device by themselves, and short ones, have a workgroup each (the rule, with both sides' times, is fa_paged_api.hip's).
// Keys are read past the caches (kStream) but by wide workgroups of small launches (the rule is there, too).
// 32 x 8 pairs of 4096 .. 16384 keys, d = 128, 1.34 GB: 212 us, 6.3 TB/s (239 through the caches); 8 pairs of 16000 23, 12 of 500 keys, d = 64, 7.8: a chain of latencies.
#include "fa_paged_decode_kernel.h"

namespace fa {

// Waves per SIMD that registers are to allow: without a bound the compiler puts the products into accumulation registers and moves them out one by one (d = 64, 32 x 8
// pairs of 4096 .. 16384 keys 135 us, with the bound 132; d = 32 75.6, 73.4).  At d = 128 LDS allows one.
constexpr int decode_bound(int head_dim, int waves) { return head_dim == 128 ? 1 : (waves == 8 ? 2 : (head_dim == 64 ? 3 : 4)); }

template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, decode_bound(D, NW)) fa_paged_decode_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[DecodeCfg<D, NW, false>::kLds];
  paged_decode<T, D, NW, false, false, NW != kDecodeWide(D)>(p, blockIdx.x, lds_raw);
}

namespace {

template <typename T, int D>
__global__ void __launch_bounds__(64 * kDecodeWide(D), decode_bound(D, kDecodeWide(D))) paged_decode_wide_stream_kernel(const PagedFwdParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[DecodeCfg<D, kDecodeWide(D), false>::kLds];
  paged_decode<T, D, kDecodeWide(D), false, false, true>(p, blockIdx.x, lds_raw);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(const PagedFwdParams p) {
  paged_decode_join<T, D, false, false>(p);
}

}  // namespace

hipError_t launch_paged_decode(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return launch_for(dtype, head_dim, [&](auto t, auto d) {
    using T = typename decltype(t)::type;
    constexpr int D = d, kWide = kDecodeWide(D), kWaves = kDecodeWaves(D);
    const auto kernel = p.wide == 2 ? paged_decode_wide_stream_kernel<T, D> : p.wide ? fa_paged_decode_kernel<T, D, kWide> : fa_paged_decode_kernel<T, D, kWaves>;
    return launch_decode(kernel, p.wide ? kWide : kWaves, paged_decode_join_kernel<T, D>, p, stream);
  });
}

}  // namespace fa
