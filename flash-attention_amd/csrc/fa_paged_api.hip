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
  bool stream;             // ... that read past the caches
  int nq_tiles, n_splits;  // chunk (fa_paged_chunk.hip)
  bool deal;
  size_t bytes;
  // a shared prefix (fa_paged_prefix_kernel.h): whether its keys are read once for all, its row tiles and key splits, and the bytes of its parts, which come first
  bool share;
  int pre_tiles, pre_splits;
  size_t pre_bytes;
  size_t whole_at;  // decode: where in the other bytes the parts of whole pairs are
};

// Workgroups of the decode kernel that are resident at once: two a compute unit at d = 128 (64 KB of tiles each), four else; over pages in 8 bits, whose workgroups
// have four waves, three at d = 64.  (us with three / four there, one new token: 2 x 12 heads of 20000 keys 20.8 / 22.6, 8 x 12 of 8000 25.5 / 26.5, 32 x 12 of 4000 .. 16000
// 105.0 / 104.2; with two 23.3, 29.2 and 106.6 where three take 22.0, 27.3 and 106.2 (bf16); d = 32 with three / four 19.6 / 21.1, 24.6 / 24.6 and 84.1 / 80.1.)
int decode_resident(int head_dim, bool k8) { return 256 * (head_dim == 128 ? 2 : k8 && head_dim == 64 ? 3 : 4); }

Plan plan_of(const fa_paged_cache& c, bool k8 = false, const fa_paged_prefix* prefix = nullptr) {
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
    bool whole = pl.wide || max_keys <= (small ? 512 : 128) || (pairs > 256 && max_keys <= (small ? 2048 : c.head_dim == 64 && pairs < 1024 ? 512 : 1024));
    // pages in 8 bits, whose tiles take half the LDS and whose line begins with wider workgroups.  us of the line / a workgroup a pair / a wide one, all lengths equal | from a
    // quarter on: d = 128, 32 pairs of 500 keys 11.3 / 10.4 / 10.2, of 1000 11.3 / 15.7 / 13.7; 128 of 1000 17.6 / 16.4 / 15.1, of 2000 21.1 / 26.7 / 22.2; 256 of 2000 30.6 /
    // 28.4 / 27.2 | 27.2 / 27.4 / 23.7, of 4000 56 / 51 / 53 | 39.5 / 47.8 / 39.4; 384 of 2000 47.8 / 44.4 / 50.7, of 4000 83 / 83 / 88; d = 64, 96 of 1000 12.2 / 12.7 /
    // 11.0, of 2000 15.1 / 21.4 / 17.1; 192 of 2000 19.2 / 21.5 / 17.8, of 4000 26.8 / 38.4 / 29.5; 384 of 1000 19.0 / 17.6 / 20.9, of 2000 26.6 / 29.2 / 32.6; d = 32, 64
    // of 1000 11.1 / 12.2 / 10.3, of 2000 12.8 / 20.4 / 16.1; 384 of 2000 26.5 / 27.7 / 23.9, of 4000 38.7 / 50.4 / 41.0
    if (k8) {
      const bool many = pairs > (small ? 512 : 256);
      pl.wide = !many && max_keys <= (pairs >= 192 ? 2048 : pairs >= 96 ? 1280 : 768);
      whole = pl.wide || max_keys <= 128 || (many && max_keys <= (c.head_dim == 64 ? 1536 : 2048));
    }
    // Keys are read once.  Past the caches that is faster where they come from memory, 32 x 8 pairs of 4096 .. 16384 keys, d = 128, 237 -> 212 us, in 8 bits 137 -> 121, 48 of 4000 22.9 -> 21.7;
    // where the caches have them from the call before it costs a little, more so in one workgroup's chain.  us through / past them, memory | caches: wide, 8 bits, 256 pairs of
    // 1000, d = 128 19.5 / 18.3 | 17.5 / 17.0, 96 of 700, d = 64 (9 MB) 10.1 / 9.9 | 9.6 / 9.7, 32 of 500 (4 MB) 10.8 / 11.0 | 10.3 / 10.8; 16 bits 256 of 1000, d = 128 29.4 / 26.3 |
    // 25.8 / 25.2, 96 of 1000, d = 64 12.4 / 11.2 | 11.0 / 11.0, 12 of 500 8.2 / 8.6 | 7.7 / 7.7.  The line always reads past them: 16 bits, 8 of 1000, d = 128 11.9 / 11.3 | 10.8 / 10.8,
    // 12 of 4000, d = 64 13.1 / 11.9 | 10.9 / 11.0, 16 of 7000 16.9 / 15.6 | 13.3 / 13.5, 8 of 6000, d = 32 10.9 / 10.4 | 9.9 / 9.9, 8 bits 8 of 2000, d = 128 11.8 / 11.4 | 10.5 / 10.5, of
    // 5000, d = 64 12.1 / 11.5 | 11.0 / 11.0
    pl.stream = pairs * max_keys * c.head_dim * (k8 ? 2 : 4) >= ((int64_t)8 << 20);
    if (!whole) {
      const int64_t units = (max_keys + fa::kDecodeUnit - 1) / fa::kDecodeUnit;
      pl.groups = (int)std::min<int64_t>(decode_resident(c.head_dim, k8), pairs * units);
      pl.bytes = (size_t)pl.groups * fa::decode_part_floats(c.head_dim) * 4;
    }
    // A shared prefix is read once for all where that is quicker.  Of 1024 keys and 8 MB saved at least: the same pages read again come out of the caches, and splitting and joining costs a
    // launch.  More than 32 rows a pair are not (8 x 4 heads, 24 tokens: 24 sequences behind 8192 keys 243 us so, 154 where each reads its own).
    const int shared = prefix ? std::min(prefix->max_prefix_len, max_keys) / c.page_size * c.page_size : 0;
    const int64_t saved = (int64_t)(c.batch - (prefix ? prefix->n_groups : 0)) * c.nheads_k * shared * c.head_dim * (k8 ? 2 : 4);
    if (shared > 0 && (prefix->always || (shared >= 1024 && saved >= ((int64_t)8 << 20)))) {
      Plan so = pl;
      so.wide = so.stream = false;
      // Row tiles of all groups, and how a prefix's keys are split: many splits are short ones, and leave as many parts to write and to read.  Of n splits the keys
      // take t = shared / n * 1.75 us / 64 (d = 128), the parts n times 8 of their bytes at 5 TB/s, beside a stream that wants them, too; together least at n =
      // sqrt(shared * 160 d / bytes of a split's parts).  At most half of the resident workgroups, and 128 keys each at least.  us with 8 / 16 / 32 splits: 32
      // sequences of 8 x 4 heads behind 8192 keys 34.2 / 33.0 / 37.9, 64 behind 16384 in 8 bits 81 / 62 / 75; of 128 / 256 / 512 keys: 3 groups of 4 x 4 heads of 3, d = 64, 3
      // tokens, behind 1667 .. 3333 15.9 / 15.2 / 20.8
      const int resident = 256 * (c.head_dim == 128 || (c.head_dim == 64 && !k8) ? 2 : 3), G = c.nheads_q / c.nheads_k;
      const int64_t all_rows = (int64_t)c.total_q * G, part = std::max<int64_t>(fa::prefix_part_rows(c.total_q, G), 4) * (c.head_dim + 3) * 4 * c.nheads_k;
      so.pre_tiles = (int)((all_rows + fa::kChunkRows - 1) / fa::kChunkRows) + prefix->n_groups - 1;
      const int64_t items = (int64_t)c.nheads_k * so.pre_tiles, best = (int64_t)std::sqrt((double)shared * 160 * c.head_dim / (double)part);
      so.pre_splits = (int)std::max<int64_t>(1, std::min<int64_t>({resident / 2 / std::max<int64_t>(items, 1), shared / 128, best, 64}));
      so.pre_bytes = fa::align16((size_t)so.pre_splits * part);
      // ... beside the line of what comes behind it, which has the other resident workgroups, and a part for each pair
      const int own = std::max(max_keys - shared, 1);
      const int64_t units = (own + fa::kDecodeUnit - 1) / fa::kDecodeUnit;
      so.groups = (int)std::min<int64_t>(std::max<int64_t>(resident - items * so.pre_splits, resident / 2), pairs * units);
      so.whole_at = (size_t)so.groups * fa::decode_part_floats(c.head_dim) * 4;
      so.bytes = so.whole_at + (size_t)pairs * rows * (c.head_dim + 4) * 4;
      // What either takes, us, fitted to 1185 pairs of times: drawn calls, and heads x sequences x prefixes of 1024 .. 100000 keys at every head dim.  The quicker one's time is exceeded by
      // 0.6 % on the average, 27 % at most, more than 5 % in one of 20; on 670 other draws by 0.7 %, 37 % at most.  (By the chain and the bytes saved alone: 2.4 %, 132 %, one of 8.)
      // Each reading its own: one launch, in which the longest sequence's workgroup decides, or the line and its join; either as the pairs' keys come in, and the distinct ones from
      // memory.  Shared: the prefix's chain of tiles beside the line's workgroups, whose every pair is a chain of its own, and splits to join.
      const double d128 = c.head_dim / 128., key = (k8 ? std::max(21.5, 25.6 * d128) : std::max(18.6, 48. * d128)) * 1e-6;
      const int waves = k8 ? (pl.wide ? fa::kDecodeWide8 : fa::kDecodeWaves8) : pl.wide ? fa::kDecodeWide(c.head_dim) : fa::kDecodeWaves(c.head_dim);
      const double keys = (double)pairs * max_keys * key + (double)prefix->n_groups * c.nheads_k * shared * c.head_dim * (k8 ? 2 : 4) * 0.064e-6;
      const double alone = whole ? 5.3 + std::max(max_keys / (29. * waves), keys) : (c.head_dim == 128 ? 14.8 : 12.2) + keys;
      const double rounds = std::max(1.0, (double)items * so.pre_splits / (resident / 2)), each = (double)pairs * units / so.groups;
      const int64_t steps = (shared + 64 * (int64_t)so.pre_splits - 1) / (64 * (int64_t)so.pre_splits);
      const double visits = each <= 1 ? 1 : 2 + std::floor((each - 1) / units);  // pairs that a workgroup of the line has to do with
      const double together = 8.1 + std::max(rounds * steps * 1.65 * std::max(0.9, d128), 7.9 * (visits - 1) + (double)pairs * own * key) + 0.133 * so.pre_splits * d128;
      // us together / alone, one new token, 300 keys of each sequence's own, 16 bits | 8:
      // 8 x 4 heads, d = 128: 2 sequences behind 2048 keys 12.4 / 14.2, 48 24.7 / 51.2 | 23.8 / 42.6; 2 behind 8192 15.4 / 20.1, 4 15.9 / 25.0 | 17.0 / 22.3, 48 32 / 133 | 32 / 108; 8 groups
      // of 4 behind 2048 26.4 / 33.8 | 29.0 / 30.8, 16 of 2 35.2 / 37.7 | 42.8 / 32.4; 2 sequences behind 100000 77 / 93 | 103 / 76.  1 x 8 heads: 4 sequences behind
      // 8192 20.2 / 15.9 | 19.9 / 14.6, 48 21.5 / 33.6 | 23.1 / 30.4, 2 behind 100000 53 / 28 | 58 / 26
      // 12 heads, d = 64: 4 behind 2048 12.1 / 13.5 | 12.5 / 14.1, 16 19.7 / 17.3 | 16.6 / 20.4, 48 29 / 38 | 26 / 41, 2 behind 8192 17.6 / 17.1 | 14.7 / 17.1, 4 17.8 / 21.6 | 14.9 / 20.8, 16 behind
      // 1024 18.6 / 12.5 | 13.5 / 13.4; 16 groups of 2 behind 2048 48 / 33 | 33 / 30 (this one told wrongly)
      // 8 heads, d = 32: 16 behind 2048 11.2 / 13.4 | 11.7 / 17.0, 8 groups of 4 15.3 / 13.7 | 17.0 / 21.9, 16 of 2 19.5 / 13.8, 16 sequences behind 8192 12.3 / 24.1 | 13.9 / 30.8
      so.share = prefix->always || together < alone;
      if (so.share) return so;
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

int check(const fa_paged_fwd_args* a, bool weights, const char* name, const fa_paged_scales* scales = nullptr) {
  FA_REQUIRE(a && a->struct_bytes == sizeof(fa_paged_fwd_args), "%s: struct size mismatch", name);
  FA_REQUIRE(a->dtype == FA_FP16 || a->dtype == FA_BF16, "%s: dtype must be fp16 or bf16", name);
  const int rc = fa::check_paged_cache(&a->cache, true, !weights, true, name, scales);
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

int check_prefix(const fa_paged_fwd_args* a, const fa_paged_prefix* x, const char* name) {
  FA_REQUIRE(x->struct_bytes == sizeof(fa_paged_prefix), "%s: prefix's struct size mismatch", name);
  FA_REQUIRE(x->n_groups > 0 && x->n_groups <= a->cache.batch && x->max_prefix_len >= 0, "%s: from one group to a group for each sequence, max_prefix_len not negative", name);
  FA_REQUIRE(x->cu_groups && x->prefix_lens && ((reinterpret_cast<uintptr_t>(x->cu_groups) | reinterpret_cast<uintptr_t>(x->prefix_lens)) & 3) == 0,
             "%s: cu_groups and prefix_lens must be there and 4-byte aligned", name);
  const int64_t rows = (int64_t)a->cache.total_q * (a->cache.nheads_q / a->cache.nheads_k);
  FA_REQUIRE(rows < ((int64_t)1 << 30) && (rows / fa::kChunkRows + x->n_groups) * a->cache.nheads_k < ((int64_t)1 << 24), "%s: too many rows", name);
  return FA_OK;
}

fa::PagedFwdParams params(const fa_paged_fwd_args* a, const fa_paged_scales* scales = nullptr) {
  fa::PagedFwdParams p{};
  p.c = fa::paged_cache(&a->cache, scales);
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

size_t fa_paged_fwd_with_workspace_bytes(const fa_paged_fwd_args* a, const fa_paged_scales* scales, const fa_paged_prefix* prefix) {
  if (!a || a->struct_bytes != sizeof(fa_paged_fwd_args) || fa::check_paged_cache(&a->cache, false, false, true, "fa_paged_fwd") != FA_OK) return 0;
  if (prefix && check_prefix(a, prefix, "fa_paged_fwd_with") != FA_OK) return 0;
  const Plan pl = plan_of(a->cache, scales != nullptr, prefix);
  return pl.pre_bytes + pl.bytes;
}

int fa_paged_fwd_with(const fa_paged_fwd_args* a, const fa_paged_scales* scales, const fa_paged_prefix* prefix) {
  const char* const name = scales || prefix ? "fa_paged_fwd_with" : "fa_paged_fwd";
  int rc = check(a, false, name, scales);
  if (!rc && prefix) rc = check_prefix(a, prefix, name);
  if (rc || a->cache.total_q == 0) return rc;
  const Plan pl = plan_of(a->cache, scales != nullptr, prefix);
  const size_t bytes = pl.pre_bytes + pl.bytes;
  if (bytes && (!a->workspace || a->workspace_bytes < bytes || !fa::aligned16(a->workspace)))
    return fa::fail(FA_ERR_WORKSPACE, "%s: needs %zu bytes of 16-byte aligned workspace", name, bytes);
  fa::PagedFwdParams p = params(a, scales);
  p.groups = pl.groups;
  p.wide = !pl.wide ? 0 : pl.stream ? 2 : 1;
  p.nq_tiles = pl.nq_tiles;
  p.n_splits = pl.n_splits;
  p.deal = pl.deal;
  p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + pl.pre_bytes);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  const int dtype = a->dtype, head_dim = a->cache.head_dim;
  if (pl.share) {
    p.c.prefix = prefix->prefix_lens;
    p.c.max_prefix = prefix->max_prefix_len;
    p.cu_groups = prefix->cu_groups;
    p.n_groups = prefix->n_groups;
    p.pre_tiles = pl.pre_tiles;
    p.pre_splits = pl.pre_splits;
    p.pre = reinterpret_cast<float*>(a->workspace);
    p.whole_part = reinterpret_cast<float*>(reinterpret_cast<char*>(p.part) + pl.whole_at);
    FA_LAUNCH((scales ? fa::launch_paged_prefix_8bit : fa::launch_paged_prefix)(p, dtype, head_dim, stream));
    return FA_OK;
  }
  if (pl.decode) FA_LAUNCH((scales ? fa::launch_paged_decode_8bit : fa::launch_paged_decode)(p, dtype, head_dim, stream));
  else FA_LAUNCH((scales ? fa::launch_paged_chunk_8bit : fa::launch_paged_chunk)(p, dtype, head_dim, stream));
  return FA_OK;
}

size_t fa_paged_fwd_workspace_bytes(const fa_paged_fwd_args* a) { return fa_paged_fwd_with_workspace_bytes(a, nullptr, nullptr); }
int fa_paged_fwd(const fa_paged_fwd_args* a) { return fa_paged_fwd_with(a, nullptr, nullptr); }

int fa_paged_key_weights(const fa_paged_fwd_args* a) {
  const int rc = check(a, true, "fa_paged_key_weights");
  if (rc || a->cache.total_q == 0) return rc;
  const fa::PagedFwdParams p = params(a);
  FA_LAUNCH(fa::launch_paged_key_weights(p, a->dtype, a->cache.head_dim, reinterpret_cast<hipStream_t>(a->stream)));
  return FA_OK;
}

}  // extern "C"
