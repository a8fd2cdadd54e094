// Where the new tokens' rows lie in a paged cache (fa_paged_append.hip, fa_paged_read.hip).
#pragma once

#include "fa_paged.h"

namespace fa {

// 16 bytes that a launch reads or writes once.  Many rows (kStream): marked as such, so that they leave the caches to what is read again.  us with / without, 20000 rows of 3 x 16 heads,
// d = 64, rows read so by the store into 16 bits 52.5 / 57.7, with attention of the chunk behind it 341 / 342, 4800 rows of 32 + 8 + 8 heads, d = 128, likewise 74.5 / 76.5, in 8 bits 82.1 /
// 83.4.  (The new q written so: 2 us less to store, and 2 more for the attention that reads it.)  Rows written so by reading, pages in the caches | in memory: 8 x 2500 rows stored and read back
// 76.7 / 79.6, 77.3 / 82.0 where the states exceed the caches; rows of 2 x 8 heads, d = 128, 8 bits, 6000 8.3 / 9.7 | 9.2 / 11.4, 15000 16.4 / 18.2 | 22.7 / 21.8, 24000 27.1 / 27.0 | 32.7 / 30.4,
// 41600 42.6 / 50.8 | 53.6 (three states in turn 58.5) / 48.7, 83200 82 / 107 | 101 / 108; 41600 in 16 bits 53.2 / 62.3 | 64.5 / 64.4.
template <bool kStream>
FA_DEVICE u32x4 ld_row16(const void* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  else return ld_global16(p);
}
template <bool kStream>
FA_DEVICE void st_row16(void* p, u32x4 v) {
  if constexpr (kStream) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
  else st_global16(p, v);
}

// Rows row0 .. row0 + ROWS - 1 of the packed new tokens, wave-uniform and all at once: their sequences (cu is non-decreasing: as many as end at or before the row; a load
// and a ballot for 64 of them), then lengths, then pages.  slot: -1 for a row that has none, page: then -1, too; pos: given_positions[row], or the slot.
template <int ROWS>
struct RowPlaces {
  int seq[ROWS], slot[ROWS], page[ROWS], pos[ROWS];
  FA_DEVICE void find(const PagedCache& c, const int32_t* given_positions, int row0) {
#pragma unroll
    for (int i = 0; i < ROWS; i++) seq[i] = 0;
    for (int at = 0; at < c.B; at += 64) {
      const int s = at + (threadIdx.x & 63);
      const int end = c.cu_q[s < c.B ? s + 1 : c.B];
#pragma unroll
      for (int i = 0; i < ROWS; i++) seq[i] += __popcll(__ballot(s < c.B && end <= row0 + i));
    }
    // (loads and what is made of them in loops of their own, without branches: the rows' loads are on their way together)
    int len[ROWS], begin[ROWS], end[ROWS];
    bool there[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int b = __builtin_amdgcn_readfirstlane(seq[i]);
      there[i] = b < c.B && row0 + i < c.total_q;  // (else: behind the last sequence)
      seq[i] = b < c.B ? b : c.B - 1;
      len[i] = ld_scalar(c.seqlens, seq[i]);
      begin[i] = ld_scalar(c.cu_q, seq[i]);
      end[i] = ld_scalar(c.cu_q, seq[i] + 1);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      slot[i] = append_slot(len[i], begin[i], end[i], row0 + i, c.max_sq, c.max_keys);
      if (!there[i]) slot[i] = -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      page[i] = ld_scalar(c.table + (int64_t)seq[i] * c.table_rs, (slot[i] < 0 ? 0 : slot[i]) >> c.page_log2);
      pos[i] = slot[i];
    }
    if (given_positions) {
#pragma unroll
      for (int i = 0; i < ROWS; i++) pos[i] = ld_scalar(given_positions, row0 + i < c.total_q ? row0 + i : c.total_q - 1);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (slot[i] < 0) page[i] = -1;
  }
};

}  // namespace fa
