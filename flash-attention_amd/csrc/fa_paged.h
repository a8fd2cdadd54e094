// The paged key / value cache as the kernels see it, and what they share: extents of a sequence, a tile's pages, staging of a tile.
#pragma once

#include "../../include/flash_attn_gfx950.h"
#include "fa_check.h"
#include "fa_paged_index.h"
#include "fa_params.h"
#include "fa_stage.h"

namespace fa {

struct PagedCache {
  char* k;
  char* v;
  int64_t k_ps, k_ss, k_hs, v_ps, v_ss, v_hs;  // page, slot and head strides in bytes
  const int32_t* table;
  int64_t table_rs;
  const int32_t* seqlens;
  const int32_t* cu_q;
  int n_pages, page_log2, max_keys;  // max_keys: most keys of a sequence that are looked at
  int B, H, HK, G;
  int total_q, max_sq;
  float* weights;      // [n_pages][HK][page size]
  int32_t* positions;
  // a cache in 8 bits (fa_paged_8bit.h): the rows' exponents, [n_pages][HK][page size]
  uint8_t* k_exps;
  uint8_t* v_exps;
  // sequences that share a prefix (fa_paged_fwd.h): how many keys of each
  const int32_t* prefix;
  int max_prefix;
};

// Everything about a cache's tensors that the entry points have in common.  needs_v / needs_q: whether v_cache / cu_seqlens_q are used.  scales: of a cache
// in 8 bits, or null.
inline int check_paged_cache(const fa_paged_cache* c, bool needs_k, bool needs_v, bool needs_q, const char* name, const fa_paged_scales* scales = nullptr) {
  FA_REQUIRE(c->head_dim == 16 || c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, "%s: head_dim must be 16, 32, 64 or 128, got %d", name,
             c->head_dim);
  FA_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
             "%s: page_size must be a power of two from 16 to 1024, got %d", name, c->page_size);
  FA_REQUIRE(c->batch > 0 && c->nheads_k > 0 && c->n_pages > 0 && c->table_cols > 0 && c->max_seqlen_k > 0, "%s: sizes must be positive", name);
  const int64_t room = (int64_t)c->table_cols * c->page_size;
  FA_REQUIRE((room < c->max_seqlen_k ? room : c->max_seqlen_k) <= ((int64_t)1 << 30), "%s: more than 2^30 keys of a sequence", name);  // (counted in 32 bits)
  FA_REQUIRE(c->nheads_k <= 65536 && c->batch <= (1 << 20) && (int64_t)c->batch * c->nheads_k < ((int64_t)1 << 24), "%s: too many sequences or heads", name);
  FA_REQUIRE(c->page_table && c->seqlens_k && c->table_row_stride >= c->table_cols, "%s: null pointer, or page table rows that overlap", name);
  FA_REQUIRE(((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->seqlens_k) | reinterpret_cast<uintptr_t>(c->cu_seqlens_q) |
               reinterpret_cast<uintptr_t>(c->key_weights) | reinterpret_cast<uintptr_t>(c->key_positions)) & 3) == 0,
             "%s: integers and weights must be 4-byte aligned", name);
  if (needs_q) {
    FA_REQUIRE(c->cu_seqlens_q && c->nheads_q > 0 && c->nheads_q % c->nheads_k == 0 && c->nheads_q / c->nheads_k <= 1024,
               "%s: nheads_q must be a multiple of nheads_k (1024 times it at most), and cu_seqlens_q be given", name);
    FA_REQUIRE(c->total_q >= 0 && c->max_seqlen_q > 0 && (int64_t)c->max_seqlen_q * (c->nheads_q / c->nheads_k) < ((int64_t)1 << 30), "%s: bad number of new tokens", name);
  }
  const auto page_ok = [](int64_t s) { return s % 8 == 0 && s >= 0 && s < ((int64_t)1 << 40); };
  if (scales) {
    FA_REQUIRE(scales->struct_bytes == sizeof(fa_paged_scales), "%s: scales' struct size mismatch", name);
    FA_REQUIRE((!needs_k || (scales->k_scales && aligned16(scales->k_scales))) && (!needs_v || (scales->v_scales && aligned16(scales->v_scales))),
               "%s: k_scales and v_scales must be there and 16-byte aligned", name);
    FA_REQUIRE((!needs_k || (c->k_page_stride % 16 == 0 && c->k_slot_stride % 16 == 0 && c->k_head_stride % 16 == 0)) &&
                   (!needs_v || (c->v_page_stride % 16 == 0 && c->v_slot_stride % 16 == 0 && c->v_head_stride % 16 == 0)),
               "%s: the strides of a cache in 8 bits must be multiples of 16 elements", name);
  }
  if (needs_k)
    FA_REQUIRE(c->k_cache && aligned16(c->k_cache) && page_ok(c->k_page_stride) && stride_ok(c->k_slot_stride) && stride_ok(c->k_head_stride),
               "%s: k_cache must be 16-byte aligned, its strides multiples of 8 elements (slots and heads below 2^24)", name);
  if (needs_v)
    FA_REQUIRE(c->v_cache && aligned16(c->v_cache) && page_ok(c->v_page_stride) && stride_ok(c->v_slot_stride) && stride_ok(c->v_head_stride),
               "%s: v_cache must be 16-byte aligned, its strides multiples of 8 elements (slots and heads below 2^24)", name);
  return FA_OK;
}

inline PagedCache paged_cache(const fa_paged_cache* c, const fa_paged_scales* scales = nullptr) {
  PagedCache p{};
  const int64_t size = scales ? 1 : 2;  // bytes of an element
  p.k = reinterpret_cast<char*>(c->k_cache);
  p.v = reinterpret_cast<char*>(c->v_cache);
  p.k_ps = c->k_page_stride * size; p.k_ss = c->k_slot_stride * size; p.k_hs = c->k_head_stride * size;
  p.v_ps = c->v_page_stride * size; p.v_ss = c->v_slot_stride * size; p.v_hs = c->v_head_stride * size;
  p.table = c->page_table;
  p.table_rs = c->table_row_stride;
  p.seqlens = c->seqlens_k;
  p.cu_q = c->cu_seqlens_q;
  p.n_pages = c->n_pages;
  p.page_log2 = __builtin_ctz((unsigned)c->page_size);
  const int64_t room = (int64_t)c->table_cols * c->page_size;
  p.max_keys = (int)(room < c->max_seqlen_k ? room : c->max_seqlen_k);
  p.B = c->batch; p.H = c->nheads_q; p.HK = c->nheads_k;
  p.G = c->nheads_k > 0 ? c->nheads_q / c->nheads_k : 0;
  p.total_q = c->total_q; p.max_sq = c->max_seqlen_q;
  p.weights = c->key_weights;
  p.positions = c->key_positions;
  if (scales) {
    p.k_exps = reinterpret_cast<uint8_t*>(scales->k_scales);
    p.v_exps = reinterpret_cast<uint8_t*>(scales->v_scales);
  }
  return p;
}

// An int32 of device memory that no kernel of the launch writes, read through the scalar cache (the index is wave-uniform): such loads are not
// among the vector loads that the staging counts.
FA_DEVICE int ld_scalar(const int32_t* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}

FA_DEVICE int paged_len(const PagedCache& c, int b) {  // keys of sequence b that are looked at
  return keys_in_reach(ld_scalar(c.seqlens, b), c.max_keys);
}
// The page that holds keys 16 g .. 16 g + 15 of a sequence (pages are 16 slots or a power of two times that), inside the pool whatever the table holds.
// Groups behind the last that is looked at stand for that one, whatever the sequence's length: a tile's pages can be asked for while that is on its way.
FA_DEVICE int page_of_group(const PagedCache& c, const int32_t* table_b, int g) {
  const int at = g >> (c.page_log2 - 4), last = (c.max_keys - 1) >> c.page_log2;
  return page_in_pool(ld_scalar(table_b, at < last ? at : last), c.n_pages);
}
// The same for a table whose first `skipped` pages are not looked at (table_b: from there on)
FA_DEVICE int page_of_group(const PagedCache& c, const int32_t* table_b, int g, int skipped) {
  const int at = g >> (c.page_log2 - 4), last = ((c.max_keys - 1) >> c.page_log2) - skipped;
  return page_in_pool(ld_scalar(table_b, at < last ? at : last), c.n_pages);
}
FA_DEVICE int slot_of_group(const PagedCache& c, int g) { return (g << 4) & ((1 << c.page_log2) - 1); }

// Stages 16 consecutive keys (or values) of a tile: such a group lies in one page, so its address is wave-uniform and a group's loads are those
// of fa_stage.h, from a base of its own.  The tile's rows are unpadded and swizzled as there (the swizzles have a period of 16 rows at most).
template <int D, int KIND, bool kStream = false>
struct GroupStager {
  static constexpr int CH = D / 8;
  static constexpr int RPI = 64 / CH < 16 ? 64 / CH : 16;  // rows per direct-to-LDS instruction (d = 16: half a wave's lanes)
  static constexpr int NI = 16 / RPI;
  static constexpr int kBytes = 16 * D * 2;
  uint32_t off[NI];  // lane: from the group's first row to the chunk that this lane fetches with instruction i
  int rl, pch;

  FA_DEVICE void init(int lane, int64_t rsb) {
    rl = lane / CH;
    pch = lane % CH;
#pragma unroll
    for (int i = 0; i < NI; i++) off[i] = (uint32_t)((i * RPI + rl) * rsb) + 16u * (uint32_t)(pch ^ tile_swz<D, KIND>(i * RPI + rl));
  }
  // last: the group's last row that may be read; rows behind it repeat it (LDS holds tensor data only, the caller masks their scores)
  FA_DEVICE void issue(const char* base, int64_t rsb, int last, unsigned char* dst) const {
    if (64 / CH > 16 && rl >= 16) return;
    if (__builtin_expect(last >= 15, 1)) {
#pragma unroll
      for (int i = 0; i < NI; i++) dma16<kStream>(base, off[i], dst + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int r = i * RPI + rl;
        dma16<kStream>(base, (uint32_t)((r < last ? r : last) * rsb) + 16u * (uint32_t)(pch ^ tile_swz<D, KIND>(r)), dst + i * 1024);
      }
    }
  }
};

}  // namespace fa
