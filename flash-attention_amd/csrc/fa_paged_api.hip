// Entry points of attention over a paged cache: checks, and how its launches are cut.
#include <algorithm>
#include <cmath>

#include "fa_paged_fwd.h"

namespace fa {
hipError_t launch_paged_key_weights(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream);  // fa_paged_weights.hip
}

namespace {

// How a forward is cut, from the call's integers alone (the lengths are on the device).
struct Plan {
  bool decode;
  int groups;              // decode (fa_paged_decode.hip)
  bool wide;               // ... eight (d = 128: four) waves a workgroup
  int nq_tiles, n_splits;  // chunk (fa_paged_chunk.hip)
  bool deal;
  size_t bytes;
};

// Workgroups of the decode kernel that are resident at once: two a compute unit at d = 128 (64 KB of tiles each), four else.
int decode_resident(int head_dim) { return 256 * (head_dim == 128 ? 2 : 4); }

Plan plan_of(const fa_paged_cache& c) {
  Plan pl{};
  const int rows = c.max_seqlen_q * (c.nheads_q / c.nheads_k);
  const int64_t pairs = (int64_t)c.batch * c.nheads_k;
  const int max_keys = (int)std::min<int64_t>(c.max_seqlen_k, (int64_t)c.table_cols * c.page_size);
  pl.decode = rows <= fa::kDecodeMaxQ;
  if (pl.decode) {
    // A pair to itself, or shares of the line of all keys and a join behind them: the join is another launch and the line's beginning a chain of loads, 14 us
    // at the least; a workgroup alone with a pair reads 26 (d = 128) or 34 keys a wave and us, and the longest sequence decides.  us of a workgroup a pair / of
    // the line, one new token, all lengths equal | from a quarter on:
    // few pairs, wide workgroups: 32 pairs of 600 keys, d = 128 13.1 / 16.5, of 1000 17.2 / 15.1; d = 64 1000 11.4 / 15.2, 2000 17.5 / 15.1; d = 32 2000 13.5 / 14.8
    // 128 pairs: d = 128 1000 19.1 / 22.5 | 20.0 / 22.4, 2000 29.9 / 32.2 | 29.5 / 26.4; d = 64 4000 29.1 / 30.2 | 26.8 / 26.0, 8000 61 / 59 | 53 / 40
    // 256 pairs: d = 128 4000 101 / 104 | 72 / 72, 8000 187 / 191 | 134 / 131; d = 64 8000 98 / 106 | 72 / 73; d = 32 8000 53 / 59 | 41 / 41
    pl.wide = pairs <= 256 && max_keys <= (pairs >= 192 ? 1024 : pairs >= 96 ? 512 : 192) * fa::kDecodeWide(c.head_dim);
    // short keys at d <= 32, more pairs than the device holds at once: the usual number of waves.  d = 32, 256 pairs of 500 8.2 / 14.7, wide 9.1; 320 of 2000 24 / 25 |
    // 22 / 22, of 4000 41 / 40 | 36 / 30; d = 64, 320 of 500 18 / 22 | 17 / 16, of 1000 29 / 26 | 26 / 22, 1024 of 1000 53 / 56 | 39 / 43; d = 128, 320 of 1000 37 / 40 |
    // 29 / 30, of 2000 71 / 71 | 54 / 53, 1024 of 1000 100 / 104 | 68 / 78
    const bool small = c.head_dim <= 32;
    if (small && max_keys <= 512) pl.wide = false;
    const bool whole = pl.wide || max_keys <= (small ? 512 : 128) || (pairs > 256 && max_keys <= (small ? 2048 : c.head_dim == 64 && pairs < 1024 ? 512 : 1024));
    if (!whole) {
      const int64_t units = (max_keys + fa::kDecodeUnit - 1) / fa::kDecodeUnit;
      pl.groups = (int)std::min<int64_t>(decode_resident(c.head_dim), pairs * units);
      pl.bytes = (size_t)pl.groups * fa::decode_part_floats(c.head_dim) * 4;
    }
    return pl;
  }
  pl.nq_tiles = (rows + fa::kChunkRows - 1) / fa::kChunkRows;
  const int64_t items = pairs * pl.nq_tiles;
  const int tiles = (max_keys + 63) / 64;
  pl.deal = pairs % 8 == 0 || pairs >= 48;  // (else one XCD would have a quarter more of them than another, or none)
  // Row tiles that do not fill the compute units share their keys: at most two workgroups a compute unit (another would be a third for some),
  // at least 256 keys each, where there are many tiles 512.  us of at least 512 keys / so: 12 heads, d = 128, 33 tokens behind 3000 25.8 / 19.0, 40 behind 460
  // 19.0 / 15.9, d = 64 18.9 / 15.9, 100 behind 900 16.8 / 15.1; 8 x 4 key heads of 16, 64 rows, 2000 keys 18.9 / 15.5; 3 x 12 heads, 100 behind 5900 27.8 / 29.9.
  // Two tiles of 512 keys, d = 64: 12.9 in one launch, 15.0 in two; 216 tiles of 700 keys 17.1 in one, 25.2 in two.  One workgroup more a tile than fits: 112 tiles,
  // d = 128 39 / 44.  256 tiles undivided 122, two each 103 (d = 128, 4000 keys).
  const int64_t n_fit = items >= 384 ? 1 : items > 256 ? 2 : 512 / items;
  const int least = items > 128 ? 8 : c.head_dim < 128 && tiles < 12 ? tiles : 4;  // tiles of 64 keys
  const int64_t n = std::min<int64_t>({n_fit, tiles / least, 64});
  pl.n_splits = n < 2 ? 1 : (int)n;
  if (pl.n_splits > 1) pl.bytes = (size_t)pl.n_splits * items * fa::kChunkRows * (c.head_dim + 3) * 4;
  return pl;
}

int check(const fa_paged_fwd_args* a, bool weights, const char* name) {
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_fwd_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  const int rc = fa::check_paged_cache(&a->cache, true, !weights, true, name);
  if (rc) return rc;
  const fa_paged_cache& c = a->cache;
  FA_REQUIRE(std::isfinite(a->softmax_scale) && a->softmax_scale > 0.f, "%s: softmax_scale must be positive and finite", name);
  const int64_t tiles = ((int64_t)c.max_seqlen_q * (c.nheads_q / c.nheads_k) + fa::kChunkRows - 1) / fa::kChunkRows;
  FA_REQUIRE((int64_t)c.batch * c.nheads_k * tiles < ((int64_t)1 << 24), "%s: too many rows", name);  // (rows times 32 float4 are counted in 32 bits of workgroups)
  if (c.total_q == 0) return FA_OK;
  FA_REQUIRE(a->q && fa::aligned16(a->q) && fa::stride_ok(a->q_row_stride) && fa::stride_ok(a->q_head_stride),
             "%s: q must be 16-byte aligned, its strides multiples of 8 elements in [0, 2^24)", name);
  if (weights) {
    FA_REQUIRE(a->softmax_lse && c.key_weights, "%s: softmax_lse and key_weights are needed", name);
    // (a tile's 64 or 128 rows are addressed from its first one's token with 32-bit offsets in bytes)
    FA_REQUIRE((c.nheads_q / c.nheads_k) * a->q_head_stride + 129 * a->q_row_stride < ((int64_t)1 << 30), "%s: q's heads of a group lie too far apart", name);
  } else {
    FA_REQUIRE(a->o && fa::aligned16(a->o) && fa::stride_ok(a->o_row_stride) && fa::stride_ok(a->o_head_stride) && a->o_row_stride >= c.head_dim &&
                   (c.nheads_q == 1 || a->o_head_stride >= c.head_dim),
               "%s: o must be 16-byte aligned, its strides multiples of 8 elements in [0, 2^24), its rows and heads apart", name);
  }
  FA_REQUIRE((reinterpret_cast<uintptr_t>(a->softmax_lse) & 3) == 0, "%s: softmax_lse must be 4-byte aligned", name);
  return FA_OK;
}

fa::PagedFwdParams params(const fa_paged_fwd_args* a) {
  fa::PagedFwdParams p{};
  p.c = fa::paged_cache(&a->cache);
  p.q = a->q;
  p.o = a->o;
  p.lse = a->softmax_lse;
  p.q_rs = a->q_row_stride; p.q_hs = a->q_head_stride; p.o_rs = a->o_row_stride; p.o_hs = a->o_head_stride;
  p.sq_r = (a->cache.max_seqlen_q + 15) / 16 * 16;
  p.causal = a->is_causal != 0;
  p.scale_log2 = a->softmax_scale * fa::kLog2e;
  return p;
}

}  // namespace

extern "C" {

size_t fa_paged_fwd_workspace_bytes(const fa_paged_fwd_args* a) {
  if (!a || a->struct_bytes != sizeof(fa_paged_fwd_args) || fa::check_paged_cache(&a->cache, false, false, true, "fa_paged_fwd") != FA_OK) return 0;
  return plan_of(a->cache).bytes;
}

int fa_paged_fwd(const fa_paged_fwd_args* a) {
  const int rc = check(a, false, "fa_paged_fwd");
  if (rc || a->cache.total_q == 0) return rc;
  const Plan pl = plan_of(a->cache);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes || !fa::aligned16(a->workspace)))
    return fa::fail(FA_ERR_WORKSPACE, "fa_paged_fwd: needs %zu bytes of 16-byte aligned workspace", pl.bytes);
  fa::PagedFwdParams p = params(a);
  p.groups = pl.groups;
  p.wide = pl.wide;
  p.nq_tiles = pl.nq_tiles;
  p.n_splits = pl.n_splits;
  p.deal = pl.deal;
  p.part = reinterpret_cast<float*>(a->workspace);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  if (pl.decode) FA_LAUNCH(fa::launch_paged_decode(p, a->dtype, a->cache.head_dim, stream));
  else FA_LAUNCH(fa::launch_paged_chunk(p, a->dtype, a->cache.head_dim, stream));
  return FA_OK;
}

int fa_paged_key_weights(const fa_paged_fwd_args* a) {
  const int rc = check(a, true, "fa_paged_key_weights");
  if (rc || a->cache.total_q == 0) return rc;
  const fa::PagedFwdParams p = params(a);
  FA_LAUNCH(fa::launch_paged_key_weights(p, a->dtype, a->cache.head_dim, reinterpret_cast<hipStream_t>(a->stream)));
  return FA_OK;
}

}  // extern "C"
