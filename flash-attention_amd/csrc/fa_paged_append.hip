// fa_paged_append: the new tokens' k and v go into their sequences' pages, k (and q, into q_out) normalised and turned on the way (fa_norm.h).
// HBM-bound for prompts (each vector read once, written once: 4.5 TB/s, of 5.3 that a copy reaches; without norm and rotation 5.1), whose workgroups
// walk over the rows; for a decode step's few rows bound by latency: the row's sequence, its
// length, its page and the store depend on each other, so the rows are loaded before any of them is asked for, and a wave finds a row's sequence
// with one load and a ballot for 64 sequences.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fa_norm.h"
#include "fa_paged.h"

namespace fa {

namespace {

struct AppendParams {
  PagedCache c;
  const void *q, *k, *v;
  void* q_out;
  const void *qw, *kw;
  const void *cos, *sin;
  const int32_t* given_positions;
  int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, qo_rs, qo_hs;  // elements
  int w_fp32, table_rows;
  float eps;
  int q_heads;  // 0 without q
  int per_row, pieces, threads, groups;
};

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(512) paged_append_kernel(const AppendParams p) {
  constexpr int CH = D / 8;
  using vec8 = typename Elem<T>::vec8;
  const int group = blockIdx.x / p.pieces, piece = blockIdx.x - group * p.pieces;
  const int j = piece * (int)blockDim.x + threadIdx.x;
  const int head = j / CH, ch = j % CH;
  const bool on = j < p.per_row;
  // heads of q, then of k, then of v
  const int part = head < p.q_heads ? 0 : (head < p.q_heads + p.c.HK ? 1 : 2);
  const int h = part == 0 ? head : (part == 1 ? head - p.q_heads : head - p.q_heads - p.c.HK);
  const T* const src = reinterpret_cast<const T*>(part == 0 ? p.q : (part == 1 ? p.k : p.v)) +
                       (int64_t)h * (part == 0 ? p.q_hs : (part == 1 ? p.k_hs : p.v_hs)) + ch * 8;
  const int64_t rs = part == 0 ? p.q_rs : (part == 1 ? p.k_rs : p.v_rs);
  const bool norm = p.kw != nullptr && part < 2, rot = p.cos != nullptr && part < 2;
  float w[8];
  if (on && norm) load_weights<T>(part == 0 ? p.qw : p.kw, p.w_fp32 != 0, ch, w);
  for (int row0 = group * ROWS; row0 < p.c.total_q; row0 += p.groups * ROWS) {
    vec8 x8[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (on && row0 + i < p.c.total_q) x8[i] = bitcast<vec8>(ld_global16(src + (int64_t)(row0 + i) * rs));
    // Where the rows go, wave-uniform and for all of them at once: their sequences (cu is non-decreasing: as many as end at or before the row; a load
    // and a ballot for 64 of them), then lengths, then pages.
    int seq[ROWS], slot[ROWS], page[ROWS], pos[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) seq[i] = 0;
    for (int at = 0; at < p.c.B; at += 64) {
      const int s = at + (threadIdx.x & 63);
      const int end = p.c.cu_q[s < p.c.B ? s + 1 : p.c.B];
#pragma unroll
      for (int i = 0; i < ROWS; i++) seq[i] += __popcll(__ballot(s < p.c.B && end <= row0 + i));
    }
    // (loads and what is made of them in loops of their own, without branches: the rows' loads are on their way together)
    int len[ROWS], begin[ROWS], end[ROWS];
    bool there[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int b = __builtin_amdgcn_readfirstlane(seq[i]);
      there[i] = b < p.c.B && row0 + i < p.c.total_q;  // (else: behind the last sequence)
      seq[i] = b < p.c.B ? b : p.c.B - 1;
      len[i] = ld_scalar(p.c.seqlens, seq[i]);
      begin[i] = ld_scalar(p.c.cu_q, seq[i]);
      end[i] = ld_scalar(p.c.cu_q, seq[i] + 1);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      slot[i] = append_slot(len[i], begin[i], end[i], row0 + i, p.c.max_sq, p.c.max_keys);
      if (!there[i]) slot[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      page[i] = ld_scalar(p.c.table + (int64_t)seq[i] * p.c.table_rs, (slot[i] < 0 ? 0 : slot[i]) >> p.c.page_log2);
      pos[i] = slot[i];
    }
    if (p.given_positions) {
#pragma unroll
      for (int i = 0; i < ROWS; i++) pos[i] = ld_scalar(p.given_positions, row0 + i < p.c.total_q ? row0 + i : p.c.total_q - 1);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (slot[i] < 0) page[i] = -1;
    // What an address has of the lane, once; the rest of it, a row's, is wave-uniform.
    typedef typename Elem<T>::vec4 vec4;
    const bool moves_only = !norm && !rot;
    const int64_t lane_to = part == 0 ? (int64_t)h * p.qo_hs * 2 + ch * 16 : (part == 1 ? h * p.c.k_hs : h * p.c.v_hs) + ch * 16;
    char* const base = part == 0 ? reinterpret_cast<char*>(p.q_out) + lane_to : (part == 1 ? p.c.k : p.c.v) + lane_to;
    vec4 c4[ROWS], s4[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int64_t row_at = (int64_t)table_row(pos[i], p.table_rows) * (D / 2);
      if (on && rot) {
        c4[i] = reinterpret_cast<const vec4*>(reinterpret_cast<const T*>(p.cos) + row_at)[ch];
        s4[i] = reinterpret_cast<const vec4*>(reinterpret_cast<const T*>(p.sin) + row_at)[ch];
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (!page_is_one(page[i], p.c.n_pages)) continue;  // (wave-uniform)
      const int at = slot[i] & ((1 << p.c.page_log2) - 1);
      const int64_t to_q = (int64_t)(row0 + i) * p.qo_rs * 2, to_k = page[i] * p.c.k_ps + at * p.c.k_ss, to_v = page[i] * p.c.v_ps + at * p.c.v_ss;
      const int64_t m0 = ((int64_t)page[i] * p.c.HK << p.c.page_log2) + at;
      if (on) {
        char* const dst = base + (part == 0 ? to_q : (part == 1 ? to_k : to_v));
        vec8 y = x8[i];
        if (!moves_only) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = (float)x8[i][e];
          if (norm) {
            const float r = inverse_rms<CH>(x, p.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * r * w[e];
          }
          if (rot) turn(x, c4[i], s4[i]);
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = (T)x[e];
        }
        st_global16(dst, bitcast<u32x4>(y));
        if (part == 1 && ch == 0) {
          const int64_t m = m0 + ((int64_t)h << p.c.page_log2);
          if (p.c.weights) p.c.weights[m] = 0.f;
          if (p.c.positions) p.c.positions[m] = pos[i];
        }
      }
    }
  }
}

template <typename T, int D>
hipError_t launch_append_d(AppendParams p, hipStream_t stream) {
  // A decode step's few rows: one a workgroup, so that as many as there are run side by side; prompts: several a thread in flight.
  constexpr int kRows = 4;  // (8 x 2500 tokens of 3 x 16 heads, d = 64, 251 MB: 55 us, two 62, eight 70: with their scalar registers full)
  const bool few = (int64_t)p.c.total_q * p.pieces <= 2048;
  const int rows = few ? 1 : kRows;
  p.groups = (p.c.total_q + rows - 1) / rows;
  // Prompts: whole workgroups a compute unit, about 20 waves of them, which walk on over the rows.  us of so many waves / as many workgroups as rows want: 20000
  // rows of 3 x 16 heads, d = 64 (six waves a workgroup, three of them a compute unit) 56 / 65, d = 32 35 / 33, 18000 of 3 x 12 40 / 49; 21000 of 40 heads 46 / 58, d = 128
  // 98 / 108; 15000 of 3 x 32, d = 128 (a row six workgroups) 158 / 153.  24 waves: 65 and 46 for the first and the third.
  if (!few) p.groups = std::min(p.groups, std::max(1, walking_workgroups(p.threads / 64, 20) / p.pieces));
  const dim3 grid((unsigned)(p.groups * p.pieces)), block((unsigned)p.threads);
  if (few) hipLaunchKernelGGL((paged_append_kernel<T, D, 1>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((paged_append_kernel<T, D, kRows>), grid, block, 0, stream, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_append(const AppendParams& p, int D, hipStream_t stream) {
  switch (D) {
    case 16: return launch_append_d<T, 16>(p, stream);
    case 32: return launch_append_d<T, 32>(p, stream);
    case 64: return launch_append_d<T, 64>(p, stream);
    case 128: return launch_append_d<T, 128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace
}  // namespace fa

extern "C" int fa_paged_append(const fa_paged_append_args* a) {
  const char* const name = "fa_paged_append";
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_append_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  const int rc = fa::check_paged_cache(&a->cache, true, true, true, name);
  if (rc) return rc;
  const fa_paged_cache& c = a->cache;
  FA_REQUIRE(c.k_slot_stride >= c.head_dim && c.v_slot_stride >= c.head_dim && (c.nheads_k == 1 || (c.k_head_stride >= c.head_dim && c.v_head_stride >= c.head_dim)) &&
                 (c.n_pages == 1 || (c.k_page_stride >= c.head_dim && c.v_page_stride >= c.head_dim)),
             "%s: the cache's slots, heads and pages must not overlap", name);
  if (c.total_q == 0) return FA_OK;
  FA_REQUIRE(a->k && a->v && fa::aligned16(a->k) && fa::aligned16(a->v) && fa::stride_ok(a->k_row_stride) && fa::stride_ok(a->k_head_stride) &&
                 fa::stride_ok(a->v_row_stride) && fa::stride_ok(a->v_head_stride),
             "%s: k and v must be 16-byte aligned, their strides multiples of 8 elements in [0, 2^24)", name);
  FA_REQUIRE((a->q == nullptr) == (a->q_out == nullptr), "%s: q and q_out come together", name);
  if (a->q)
    FA_REQUIRE(fa::aligned16(a->q) && fa::aligned16(a->q_out) && fa::stride_ok(a->q_row_stride) && fa::stride_ok(a->q_head_stride) &&
                   fa::stride_ok(a->q_out_row_stride) && fa::stride_ok(a->q_out_head_stride) && a->q_out_row_stride >= c.head_dim &&
                   (c.nheads_q == 1 || a->q_out_head_stride >= c.head_dim),
               "%s: q and q_out must be 16-byte aligned, their strides multiples of 8 elements in [0, 2^24), written rows and heads apart", name);
  FA_REQUIRE(!a->q || (a->q_weight == nullptr) == (a->k_weight == nullptr), "%s: q_weight and k_weight come together", name);
  FA_REQUIRE(!a->k_weight || a->weight_dtype == a->dtype || a->weight_dtype == FA_FP32, "%s: weights must be of the tensors' dtype or fp32", name);
  FA_REQUIRE(a->eps >= 0.f, "%s: eps must not be negative", name);
  FA_REQUIRE((a->cos_table == nullptr) == (a->sin_table == nullptr) && (!a->cos_table || a->table_rows >= 1), "%s: cos_table and sin_table come together, with rows", name);
  FA_REQUIRE(((reinterpret_cast<uintptr_t>(a->cos_table) | reinterpret_cast<uintptr_t>(a->sin_table)) & 7) == 0, "%s: tables must be 8-byte aligned", name);
  fa::AppendParams p{};
  p.c = fa::paged_cache(&c);
  p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->q_out;
  p.qw = a->q_weight; p.kw = a->k_weight;
  p.cos = a->cos_table; p.sin = a->sin_table;
  p.given_positions = a->positions;
  p.q_rs = a->q_row_stride; p.q_hs = a->q_head_stride; p.k_rs = a->k_row_stride; p.k_hs = a->k_head_stride;
  p.v_rs = a->v_row_stride; p.v_hs = a->v_head_stride; p.qo_rs = a->q_out_row_stride; p.qo_hs = a->q_out_head_stride;
  p.w_fp32 = a->weight_dtype == FA_FP32;
  p.table_rows = a->table_rows;
  p.eps = a->eps;
  p.q_heads = a->q ? c.nheads_q : 0;
  p.per_row = (p.q_heads + 2 * c.nheads_k) * (c.head_dim / 8);
  // a row's vectors go to one workgroup of whole waves if at most 512 threads, else to workgroups of 256
  p.threads = p.per_row <= 512 ? (p.per_row + 63) / 64 * 64 : 256;
  p.pieces = (p.per_row + p.threads - 1) / p.threads;
  FA_REQUIRE(c.total_q < (1 << 30) && (int64_t)c.total_q * p.pieces < ((int64_t)1 << 31), "%s: too many rows", name);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  FA_LAUNCH(a->dtype == FA_FP16 ? fa::launch_append<_Float16>(p, c.head_dim, stream) : fa::launch_append<__bf16>(p, c.head_dim, stream));
  return FA_OK;
}
