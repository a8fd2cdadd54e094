// fa_paged_read: the new tokens' (or whole sequences') keys and values out of their pages, packed, in 16 bits: the counterpart of fa_paged_append, whose places they
// lie in.  HBM-bound (41600 rows of 2 x 8 heads, d = 128, from memory: 8 bits 256 MB in 54 us, 4.8 TB/s, to 58; 16 bits 341 MB in 64.5, 5.3); what rows in 8 bits stand for is exact in 16, so nothing is rounded.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "fa_norm.h"
#include "fa_paged_8bit.h"
#include "fa_paged_rows.h"

namespace fa {

namespace {

struct ReadParams {
  PagedCache c;
  void *k, *v;
  int64_t k_rs, k_hs, v_rs, v_hs;  // bytes
  int per_row, pieces, threads, groups;
};

// A thread has 8 elements of a row's place (key or value, head, chunk) and walks over rows.  (16 elements of 8 bits, 32 bytes out: 61 us for 46000 rows of 2 x 8 heads,
// d = 128: the lanes' stores leave gaps that another instruction fills.)
template <typename T, int D, int ROWS, bool k8>
__global__ void __launch_bounds__(512) paged_read_kernel(const ReadParams p) {
  constexpr int CH = D / 8, kBytes = k8 ? 8 : 16;
  using Chunk = std::conditional_t<k8, u32x2, u32x4>;
  const int group = blockIdx.x / p.pieces, piece = blockIdx.x - group * p.pieces;
  const int j = piece * (int)blockDim.x + threadIdx.x;
  const int head = j / CH, ch = j % CH;
  const bool on = j < p.per_row, second = head >= p.c.HK;
  const int h = second ? head - p.c.HK : head;
  const char* const src = (second ? p.c.v + h * p.c.v_hs : p.c.k + h * p.c.k_hs) + ch * kBytes;
  char* const dst = reinterpret_cast<char*>(second ? p.v : p.k) + h * (second ? p.v_hs : p.k_hs) + ch * 16;
  const int64_t to_row = second ? p.v_rs : p.k_rs;
  const uint8_t* const exps = second ? p.c.v_exps : p.c.k_exps;
  for (int row0 = group * ROWS; row0 < p.c.total_q; row0 += p.groups * ROWS) {
    RowPlaces<ROWS> at;
    at.find(p.c, nullptr, row0);
    Chunk x[ROWS];
    int e[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int page = page_in_pool(at.page[i], p.c.n_pages), slot = at.slot[i] & ((1 << p.c.page_log2) - 1);
      const int64_t from_k = page * p.c.k_ps + slot * p.c.k_ss, from_v = page * p.c.v_ps + slot * p.c.v_ss;
      x[i] = Chunk{};
      e[i] = 127;
      if (on && at.slot[i] >= 0) {
        x[i] = *reinterpret_cast<const Chunk*>(src + (second ? from_v : from_k));
        if constexpr (k8) e[i] = exps[((int64_t)page * p.c.HK + h << p.c.page_log2) + slot];
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (!on || row0 + i >= p.c.total_q) continue;
      char* const to = dst + (int64_t)(row0 + i) * to_row;
      if constexpr (k8) {
        st_row16<(ROWS > 1)>(to, bitcast<u32x4>(dequant8<T>(x[i], power_of_two(e[i]))));
      } else {
        st_row16<(ROWS > 1)>(to, x[i]);
      }
    }
  }
}

template <typename T, int D, bool k8>
hipError_t launch_read_d(ReadParams p, hipStream_t stream) {
  p.per_row = 2 * p.c.HK * (D / 8);
  p.threads = p.per_row <= 512 ? (p.per_row + 63) / 64 * 64 : 256;
  p.pieces = (p.per_row + p.threads - 1) / p.threads;
  constexpr int kRows = 4;
  const bool few = (int64_t)p.c.total_q * p.pieces <= 2048;
  const int rows = few ? 1 : kRows;
  p.groups = (p.c.total_q + rows - 1) / rows;
  if (!few) p.groups = std::min(p.groups, std::max(1, walking_workgroups(p.threads / 64, 28) / p.pieces));
  const dim3 grid((unsigned)(p.groups * p.pieces)), block((unsigned)p.threads);
  if (few) hipLaunchKernelGGL((paged_read_kernel<T, D, 1, k8>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((paged_read_kernel<T, D, kRows, k8>), grid, block, 0, stream, p);
  return hipGetLastError();
}
template <typename T, bool k8>
hipError_t launch_read(const ReadParams& p, int D, hipStream_t stream) {
  switch (D) {
    case 16: return launch_read_d<T, 16, k8>(p, stream);
    case 32: return launch_read_d<T, 32, k8>(p, stream);
    case 64: return launch_read_d<T, 64, k8>(p, stream);
    case 128: return launch_read_d<T, 128, k8>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace
}  // namespace fa

extern "C" int fa_paged_read(const fa_paged_read_args* a, const fa_paged_scales* scales) {
  const char* const name = "fa_paged_read";
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_read_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  fa_paged_cache c = a->cache;
  c.nheads_q = c.nheads_k;  // (there are no queries here)
  c.max_seqlen_q = c.total_q > 0 ? c.total_q : 1;
  const int rc = fa::check_paged_cache(&c, true, true, true, name, scales);
  if (rc) return rc;
  if (c.total_q == 0) return FA_OK;
  FA_REQUIRE(a->k_out && a->v_out && fa::aligned16(a->k_out) && fa::aligned16(a->v_out) && fa::stride_ok(a->k_row_stride) && fa::stride_ok(a->k_head_stride) &&
                 fa::stride_ok(a->v_row_stride) && fa::stride_ok(a->v_head_stride) && a->k_row_stride >= c.head_dim && a->v_row_stride >= c.head_dim &&
                 (c.nheads_k == 1 || (a->k_head_stride >= c.head_dim && a->v_head_stride >= c.head_dim)),
             "%s: k_out and v_out must be 16-byte aligned, their strides multiples of 8 elements in [0, 2^24), their rows and heads apart", name);
  fa::ReadParams p{};
  p.c = fa::paged_cache(&c, scales);
  p.k = a->k_out; p.v = a->v_out;
  p.k_rs = a->k_row_stride * 2; p.k_hs = a->k_head_stride * 2; p.v_rs = a->v_row_stride * 2; p.v_hs = a->v_head_stride * 2;
  FA_REQUIRE(c.total_q < (1 << 30) && (int64_t)c.total_q * ((2 * c.nheads_k * (c.head_dim / 8) + 255) / 256) < ((int64_t)1 << 31), "%s: too many rows", name);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  if (scales) FA_LAUNCH(a->dtype == FA_FP16 ? (fa::launch_read<_Float16, true>(p, c.head_dim, stream)) : (fa::launch_read<__bf16, true>(p, c.head_dim, stream)));
  else FA_LAUNCH(a->dtype == FA_FP16 ? (fa::launch_read<_Float16, false>(p, c.head_dim, stream)) : (fa::launch_read<__bf16, false>(p, c.head_dim, stream)));
  return FA_OK;
}
