// Attention of new tokens over a paged cache: what its two kernels (fa_paged_decode.hip: at most 32 rows a key head; fa_paged_chunk.hip: any
// number) and the entry points (fa_paged_api.hip) share.
//
// Rows.  The query heads of a group read the same keys: the G heads of the Lq new tokens of a sequence are G * Lq rows of one product, row r being
// head r % G of token r / G, so that a key head's keys are read once for all of them.  Row r sees the keys below limit(r) = Lk - Lq + r / G + 1
// under the causal mask (aligned at the end), Lk else; a limit of 0 or less: nothing, o = 0 and lse = -inf.
#pragma once

#include "fa_paged.h"

namespace fa {

struct PagedFwdParams {
  PagedCache c;
  const void* q;
  void* o;
  float* lse;  // null: not wanted
  int64_t q_rs, q_hs, o_rs, o_hs;  // elements
  int sq_r;
  int causal;
  float scale_log2;
  // decode: the workgroups that share the line of units (0: a workgroup a pair), and whether they are wide.  chunk: query tiles and key splits
  int groups, wide;
  int nq_tiles, n_splits, deal;
  float* part;  // partial results
};

// Partial results of a row: its output before the division, the maximum m of its scores (before scaling), the sum l of the probabilities as they are
// rounded for the product with V, and the sum u of the unrounded ones, all with respect to m.  o = sum o_s 2^(m_s - m) / sum l_s 2^(m_s - m): numerator
// and denominator carry the same rounding; lse comes from u.
struct PartRow {
  float m, l, u;
};

// Four elements of a row, joined from parts.
struct JoinedRow {
  PartRow a{-INFINITY, 0.f, 0.f};
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  FA_DEVICE void add(PartRow x, f32x4 xo, float cs) {
    const float top = fmaxf(a.m, x.m), ref = top == -INFINITY ? 0.f : top;
    const float fa = fast_exp2((a.m - ref) * cs), fb = fast_exp2((x.m - ref) * cs);
    a = PartRow{top, a.l * fa + x.l * fb, a.u * fa + x.u * fb};
    o = o * fa + xo * fb;
  }
  // A workgroup's `lanes` (a power of two) partial joins of each row, kCols threads apart, in a fixed order; lane 0 has the result.
  template <int kCols>
  FA_DEVICE void across(int lane, int lanes, float cs, f32x4* os, PartRow* ms) {
    for (int half = lanes / 2; half > 0; half /= 2) {
      os[threadIdx.x] = o;
      ms[threadIdx.x] = a;
      __syncthreads();
      if (lane < half) add(ms[threadIdx.x + half * kCols], os[threadIdx.x + half * kCols], cs);
      __syncthreads();
    }
  }
};

FA_DEVICE bool paged_rows(const PagedCache& c, int b, int* begin, int* len) {  // the new tokens of sequence b
  const int s = ld_scalar(c.cu_q, b), e = ld_scalar(c.cu_q, b + 1);
  if (s < 0 || e <= s || e > c.total_q) return false;
  *begin = s;
  *len = e - s < c.max_sq ? e - s : c.max_sq;
  return true;
}

template <typename T>
FA_DEVICE void store_row_piece(const PagedFwdParams& p, int q_begin, int h, int r, int d0, f32x4 o) {
  const int t = r / p.c.G, g = r - t * p.c.G;
  T* const op = reinterpret_cast<T*>(p.o) + (int64_t)(q_begin + t) * p.o_rs + (int64_t)(h * p.c.G + g) * p.o_hs + d0;
  *reinterpret_cast<typename Elem<T>::vec4*>(op) = cvt4<T>(o);
}
FA_DEVICE void store_lse(const PagedFwdParams& p, int b, int h, int r, float lse) {
  if (p.lse == nullptr) return;
  const int t = r / p.c.G, g = r - t * p.c.G;
  p.lse[((int64_t)b * p.c.H + h * p.c.G + g) * p.sq_r + t] = lse;
}
FA_DEVICE float lse_of(float m, float u, float cs) { return u > 0.f ? (m * cs + fast_log2(u)) * kLn2 : -INFINITY; }

// ---- decode: keys are dealt out in units of kUnit; a pair (sequence, key head) has ceil(keys / kUnit), one at least, so that its rows are written
constexpr int kDecodeUnit = 128;
constexpr int kPartRows = 32;
// Waves of a workgroup that has a pair to itself where pairs about fill the device: as many as their tiles' LDS allows.
constexpr int kDecodeWide(int head_dim) { return head_dim == 128 ? 4 : 8; }

// floats of a workgroup's two partial results: [2][32][D] outputs, [2][3][32] m, l, u
inline size_t decode_part_floats(int D) { return 2 * (size_t)kPartRows * (D + 3); }

hipError_t launch_paged_decode(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
hipError_t launch_paged_chunk(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
constexpr int kChunkRows = 128;  // rows of a workgroup of the chunk kernel

}  // namespace fa
