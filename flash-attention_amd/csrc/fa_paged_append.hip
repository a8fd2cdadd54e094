// fa_paged_append: the new tokens' k and v go into their sequences' pages, k (and q, into q_out) normalised and turned on the way (fa_norm.h).
// HBM-bound for prompts (each vector read once, written once: 4.8 TB/s, of 5.4 that a copy reaches; into 8 bits 4.1), whose workgroups
// walk over the rows; for a decode step's few rows bound by latency: the row's sequence, its
// length, its page and the store depend on each other, so the rows are loaded before any of them is asked for, and a wave finds a row's sequence
// with one load and a ballot for 64 sequences.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fa_norm.h"
#include "fa_paged_8bit.h"
#include "fa_paged_rows.h"

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

// kQuant: into pages in 8 bits (fa_paged_8bit.h), k straight from 32 bits
template <typename T, int D, int ROWS, bool kQuant>
FA_DEVICE void paged_append(const AppendParams p) {
  constexpr int CH = D / 8;
  using vec8 = typename Elem<T>::vec8;
  const int group = blockIdx.x / p.pieces, piece = blockIdx.x - group * p.pieces;
  const int j = piece * (int)blockDim.x + threadIdx.x;
  const bool on = j < p.per_row;  // (a thread without a place loads what the last one does, so that no branch stands between the rows' loads)
  const int head = (on ? j : p.per_row - 1) / CH, ch = (on ? j : p.per_row - 1) % CH;
  // heads of q, then of k, then of v
  const int part = head < p.q_heads ? 0 : (head < p.q_heads + p.c.HK ? 1 : 2);
  const int h = part == 0 ? head : (part == 1 ? head - p.q_heads : head - p.q_heads - p.c.HK);
  const T* const src = reinterpret_cast<const T*>(part == 0 ? p.q : (part == 1 ? p.k : p.v)) +
                       (int64_t)h * (part == 0 ? p.q_hs : (part == 1 ? p.k_hs : p.v_hs)) + ch * 8;
  const int64_t rs = part == 0 ? p.q_rs : (part == 1 ? p.k_rs : p.v_rs);
  const bool norm = p.kw != nullptr && part < 2, rot = p.cos != nullptr && part < 2;
  float w[8];
  if (norm) load_weights<T>(part == 0 ? p.qw : p.kw, p.w_fp32 != 0, ch, w);
#pragma unroll
  for (int e = 0; e < 8; e++) asm volatile("" : "+v"(w[e]));  // (waited for here: in the loop it would be the last trip's stores that are waited for)
  for (int row0 = group * ROWS; row0 < p.c.total_q; row0 += p.groups * ROWS) {
    vec8 x8[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) x8[i] = bitcast<vec8>(ld_row16<(ROWS > 1)>(src + (int64_t)(row0 + i < p.c.total_q ? row0 + i : p.c.total_q - 1) * rs));
    RowPlaces<ROWS> at;
    at.find(p.c, p.given_positions, row0);
    // (the rows have come in with what that looked up; said here, since on paths that drop a row its load would count as under way, and the next trip's
    // loads would wait for all of this one's stores)
#pragma unroll
    for (int i = 0; i < ROWS; i++) asm volatile("" : "+v"(x8[i]));
    // What an address has of the lane, once; the rest of it, a row's, is wave-uniform.
    typedef typename Elem<T>::vec4 vec4;
    const bool moves_only = !norm && !rot;
    const int chunk = kQuant ? 8 : 16;  // bytes of a lane's elements in the cache
    const int64_t lane_to = part == 0 ? (int64_t)h * p.qo_hs * 2 + ch * 16 : (part == 1 ? h * p.c.k_hs : h * p.c.v_hs) + ch * chunk;
    char* const base = part == 0 ? reinterpret_cast<char*>(p.q_out) + lane_to : (part == 1 ? p.c.k : p.c.v) + lane_to;
    vec4 c4[ROWS], s4[ROWS];
    if (rot) {
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const int64_t row_at = (int64_t)table_row(at.pos[i], p.table_rows) * (D / 2);
        c4[i] = reinterpret_cast<const vec4*>(reinterpret_cast<const T*>(p.cos) + row_at)[ch];
        s4[i] = reinterpret_cast<const vec4*>(reinterpret_cast<const T*>(p.sin) + row_at)[ch];
      }
#pragma unroll
      for (int i = 0; i < ROWS; i++) asm volatile("" : "+v"(c4[i]), "+v"(s4[i]));  // (all of them before the first store, behind which a load would wait for it)
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (!page_is_one(at.page[i], p.c.n_pages)) continue;  // (wave-uniform)
      const int slot = at.slot[i] & ((1 << p.c.page_log2) - 1);
      const int64_t to_q = (int64_t)(row0 + i) * p.qo_rs * 2, to_k = at.page[i] * p.c.k_ps + slot * p.c.k_ss, to_v = at.page[i] * p.c.v_ps + slot * p.c.v_ss;
      const int64_t m0 = ((int64_t)at.page[i] * p.c.HK << p.c.page_log2) + slot;
      if (on) {
        char* const dst = base + (part == 0 ? to_q : (part == 1 ? to_k : to_v));
        vec8 y = x8[i];
        float x[8];
        if (!moves_only || kQuant) {
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = (float)x8[i][e];
        }
        if (!moves_only) {
          if (norm) {
            const float r = inverse_rms<CH>(x, p.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * r * w[e];
          }
          if (rot) turn(x, c4[i], s4[i]);
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = (T)x[e];
        }
        const int64_t m = m0 + ((int64_t)h << p.c.page_log2);
        if constexpr (kQuant) {
          if (part == 0) {
            st_global16(dst, bitcast<u32x4>(y));
          } else {
            const int byte = row_exponent<T>(vector_max<CH>(finite_top(x)));
            *reinterpret_cast<u32x2*>(dst) = quant8<T>(x, byte);
            if (ch == 0) (part == 1 ? p.c.k_exps : p.c.v_exps)[m] = (uint8_t)byte;
          }
        } else {
          st_global16(dst, bitcast<u32x4>(y));
        }
        if (part == 1 && ch == 0) {
          if (p.c.weights) p.c.weights[m] = 0.f;
          if (p.c.positions) p.c.positions[m] = at.pos[i];
        }
      }
    }
  }
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(512) paged_append_kernel(const AppendParams p) {
  paged_append<T, D, ROWS, false>(p);
}
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(512) paged_append_8bit_kernel(const AppendParams p) {
  paged_append<T, D, ROWS, true>(p);
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
  if (p.c.k_exps) {
    if (few) hipLaunchKernelGGL((paged_append_8bit_kernel<T, D, 1>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_append_8bit_kernel<T, D, kRows>), grid, block, 0, stream, p);
    return hipGetLastError();
  }
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

extern "C" int fa_paged_append(const fa_paged_append_args* a) { return fa_paged_append_with(a, nullptr); }

extern "C" int fa_paged_append_with(const fa_paged_append_args* a, const fa_paged_scales* scales) {
  const char* const name = scales ? "fa_paged_append_with" : "fa_paged_append";
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_append_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  const int rc = fa::check_paged_cache(&a->cache, true, true, true, name, scales);
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
  p.c = fa::paged_cache(&c, scales);
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
