// Attention of new tokens over a paged cache: what its two kernels (fa_paged_decode.hip: at most 32 rows a key head; fa_paged_chunk.hip: any
// number) and the entry points (fa_paged_api.hip) share.
//
// Rows.  The query heads of a group read the same keys: the G heads of the Lq new tokens of a sequence are G * Lq rows of one product, row r being
// head r % G of token r / G, so that a key head's keys are read once for all of them.  Row r sees the keys below limit(r) = Lk - Lq + r / G + 1
// under the causal mask (aligned at the end), Lk else; a limit of 0 or less: nothing, o = 0 and lse = -inf.
//
// Shared prefixes.  The sequences of a group list the same pages for their first prefix[b] keys (whole pages), which all their new tokens see.  To those keys the
// group's rows are one product, G times the tokens of all its sequences, so that the keys are read once per 128 of them, as if the group were one sequence without a
// mask; the sequences' own keys are attended as ever; both leave partial results, which a second kernel joins (fa_paged_prefix_kernel.h).  At most 32 rows a pair: with
// more of them products bound both ways, and reading a key once more costs nothing.
#pragma once

#include <type_traits>

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
  // decode: the workgroups that share the line of units (0: a workgroup a pair), and whether they are wide (2: and read past the caches).  chunk: query tiles and key splits
  int groups, wide;
  int nq_tiles, n_splits, deal;
  float* part;  // partial results
  // shared prefixes: groups of sequences (cu_groups[g] .. cu_groups[g + 1]), the splits of a prefix's keys, the row tiles that there can be, and the parts:
  // [split][key head][G * total_q rows, up to a multiple of four][D], m, l and u behind all of them
  const int32_t* cu_groups;
  int n_groups, pre_splits, pre_tiles;
  float* pre;
  float* whole_part;  // decode: the part of a pair that one workgroup has whole, for each pair
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

// Rows of a key head in a prefix's parts: those of the call, up to a multiple of four, since a split's (D + 3) floats a row are to begin at 16 bytes, too
__host__ __device__ __forceinline__ int64_t prefix_part_rows(int total_q, int G) { return ((int64_t)total_q * G + 3) / 4 * 4; }
// The keys of sequence b that its group shares: what comes in front of its own ones
template <bool kPrefix>
FA_DEVICE int first_own(const PagedCache& c, int b) {
  if constexpr (!kPrefix) return 0;
  else return shared_keys(ld_scalar(c.prefix, b), c.max_prefix, c.max_keys, c.page_log2);
}
template <bool kPrefix>
FA_DEVICE int own_len(const PagedCache& c, int b) {
  if constexpr (!kPrefix) return paged_len(c, b);
  const int n = paged_len(c, b) - first_own<kPrefix>(c, b);
  return n > 0 ? n : 0;
}
// Adds the prefix's parts lane, lane + lanes, .. of a row (of all the call's rows of key head h) to x, several at a time, whose loads are on their way together and whose
// maxima are compared first.  A part's maximum is one of scores before scaling; `unit` brings it to x's units.
template <int D>
FA_DEVICE void add_prefix(const PagedFwdParams& p, JoinedRow* x, int h, int64_t row, int d0, float cs, float unit, int lane = 0, int lanes = 1) {
  constexpr int kBatch = 4;
  const int64_t rows = prefix_part_rows(p.c.total_q, p.c.G), all = (int64_t)p.c.HK * rows, at = (int64_t)h * rows + row;
  const float* from = p.pre + (int64_t)lane * all * (D + 3);
  const int64_t step = (int64_t)lanes * all * (D + 3);
  for (int i = lane; i < p.pre_splits; i += kBatch * lanes) {
    PartRow m[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const float* const ml = from + all * D + at * 3;
      m[j] = PartRow{ml[0] * unit, ml[1], ml[2]};
      o[j] = *reinterpret_cast<const f32x4*>(from + at * D + d0);
      if (i + (j + 1) * lanes < p.pre_splits) from += step;  // (behind the last one: that one again, and not counted)
    }
#pragma unroll
    for (int j = 1; j < kBatch; j++)
      if (i + j * lanes >= p.pre_splits) m[j] = PartRow{-INFINITY, 0.f, 0.f}, o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = x->a.m;
#pragma unroll
    for (int j = 0; j < kBatch; j++) top = fmaxf(top, m[j].m);
    const float ref = top == -INFINITY ? 0.f : top * cs, f = fast_exp2(x->a.m * cs - ref);
    x->a = PartRow{top, x->a.l * f, x->a.u * f};
    x->o = x->o * f;
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const float w = fast_exp2(m[j].m * cs - ref);
      x->a.l = __builtin_fmaf(m[j].l, w, x->a.l);
      x->a.u = __builtin_fmaf(m[j].u, w, x->a.u);
      x->o = x->o + o[j] * w;
    }
  }
}

FA_DEVICE bool paged_rows(const PagedCache& c, int b, int* begin, int* len) {  // the new tokens of sequence b
  const int s = ld_scalar(c.cu_q, b), e = ld_scalar(c.cu_q, b + 1);
  if (s < 0 || e <= s || e > c.total_q) return false;
  *begin = s;
  *len = e - s < c.max_sq ? e - s : c.max_sq;
  return true;
}

// Group g: its first sequence, where its new tokens begin, and how many all its sequences have
FA_DEVICE bool group_rows(const PagedFwdParams& p, int g, int* b, int* begin, int* tokens) {
  const int b0 = p.cu_groups[g], b1 = p.cu_groups[g + 1];
  if (b0 < 0 || b1 <= b0 || b1 > p.c.B) return false;
  const int s = p.c.cu_q[b0], e = p.c.cu_q[b1];
  if (s < 0 || e <= s || e > p.c.total_q) return false;
  *b = b0;
  *begin = s;
  *tokens = e - s;
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
// ... over pages in 8 bits, whose tiles take half the LDS, and of one that has its share of the line
constexpr int kDecodeWide8 = 8;
constexpr int kDecodeWaves8 = 4;
// ... beside the workgroups of a shared prefix, which have four: two at d = 128 in 16 bits, the other two end at once, so that two workgroups' tiles fit a compute unit
constexpr int kDecodeBeside(int head_dim, bool k8) { return !k8 && head_dim == 128 ? 2 : 4; }

// A row's part is D elements, m, l and u and one float more, so that rows begin at 16 bytes; floats of a workgroup's two parts
inline size_t decode_part_floats(int D) { return 2 * (size_t)kPartRows * (D + 4); }

hipError_t launch_paged_decode(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
hipError_t launch_paged_chunk(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
// of a cache in 8 bits
hipError_t launch_paged_decode_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
hipError_t launch_paged_chunk_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
// of sequences that share a prefix
hipError_t launch_paged_prefix(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
hipError_t launch_paged_prefix_8bit(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);
constexpr int kChunkRows = 128;  // rows of a workgroup of the chunk kernel
// ... whose splits' parts, in fp32 whatever the cache holds, are joined
hipError_t launch_paged_chunk_join(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);

// launch(Type<T>{}, std::integral_constant<int, D>{}) with the element type of a dtype's code and the head dim
template <typename T>
struct Type {
  using type = T;
};
template <typename F>
hipError_t launch_for(int dtype, int head_dim, const F& launch) {
  const auto of_type = [&](auto t) {
    switch (head_dim) {
      case 16: return launch(t, std::integral_constant<int, 16>{});
      case 32: return launch(t, std::integral_constant<int, 32>{});
      case 64: return launch(t, std::integral_constant<int, 64>{});
      case 128: return launch(t, std::integral_constant<int, 128>{});
      default: return hipErrorInvalidValue;
    }
  };
  return dtype == 0 ? of_type(Type<_Float16>{}) : of_type(Type<__bf16>{});
}

}  // namespace fa
