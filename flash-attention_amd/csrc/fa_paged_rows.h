// Where the new tokens' rows lie in a paged cache (fa_paged_append.hip, fa_paged_read.hip).
#pragma once

#include "fa_paged.h"

namespace fa {

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
