// Keys of ragged sequences dealt out evenly (fa_paged_decode.hip, fa_paged_weights.hip).  Lengths are known on the device only: all units of kDecodeUnit keys of all
// pairs (sequence, key head) are laid out in one line, pair after pair, and each of the launch's workgroups takes an equal share of it - the end of one
// pair, some whole pairs, the beginning of another.  Every wave finds its share by itself, from prefix sums over 64 sequences at a time.
#pragma once

#include "fa_paged_fwd.h"

namespace fa {

template <int N>
FA_DEVICE void wait_vmcnt() {  // at most N of this wave's global loads (direct-to-LDS ones included) are still outstanding
  static_assert(N < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
}

// The line of units.  Sequence b has HK pairs of units(b) each; a sequence without new tokens has none.  kPrefix: of its own keys, behind those that its group shares.
template <bool kPrefix = false>
FA_DEVICE int units_of(const PagedCache& c, int b) {
  int keys = keys_in_reach(c.seqlens[b], c.max_keys);
  if constexpr (kPrefix) keys -= shared_keys(c.prefix[b], c.max_prefix, c.max_keys, c.page_log2);
  const int s = c.cu_q[b], e = c.cu_q[b + 1];
  if (s < 0 || e <= s || e > c.total_q) return 0;
  return keys <= kDecodeUnit ? 1 : (keys + kDecodeUnit - 1) / kDecodeUnit;
}
// Units of 64 sequences from `first` on as inclusive sums over the lanes; the same in every wave
template <bool kPrefix = false>
FA_DEVICE int unit_sums(const PagedCache& c, int first) {
  const int b = first + (threadIdx.x & 63);
  return wave_prefix_sum(b < c.B ? units_of<kPrefix>(c, b) : 0);
}
// (sums0: the first 64 sequences' sums, made once)
template <bool kPrefix = false>
FA_DEVICE int64_t all_units(const PagedCache& c, int sums0) {
  int64_t n = __builtin_amdgcn_readlane(sums0, 63);
  for (int first = 64; first < c.B; first += 64) n += __builtin_amdgcn_readlane(unit_sums<kPrefix>(c, first), 63);
  return n * c.HK;
}
struct Spot {  // a unit of the line
  int b, h, unit, units;  // units: of each pair of sequence b
};
template <bool kPrefix = false>
FA_DEVICE Spot spot_of(const PagedCache& c, int64_t u, int sums0) {
  int64_t before = 0;
  for (int first = 0; first < c.B; first += 64) {
    const int sums = first == 0 ? sums0 : unit_sums<kPrefix>(c, first);
    const int all = __builtin_amdgcn_readlane(sums, 63);
    if (u < before + (int64_t)all * c.HK) {
      const int64_t rest = u - before;
      const int lane = __popcll(__ballot((int64_t)sums * c.HK <= rest));  // sequences that end before the unit
      const int upto = lane > 0 ? __builtin_amdgcn_readlane(sums, lane > 0 ? lane - 1 : 0) : 0;
      const int units = __builtin_amdgcn_readlane(sums, lane) - upto;
      const int in_seq = (int)(rest - (int64_t)upto * c.HK);
      return Spot{first + lane, in_seq / units, in_seq % units, units};
    }
    before += (int64_t)all * c.HK;
  }
  return Spot{c.B, 0, 0, 1};
}
// Workgroups that share the line, and the first unit of workgroup w
FA_DEVICE int sharers(const PagedFwdParams& p, int64_t units) {
  return units >= p.groups ? p.groups : units > 0 ? (int)units : 1;
}
// (a quotient of numbers that are not negative: 64 bits of division are some hundred instructions, and these stand in front of everything)
FA_DEVICE int64_t quotient(int64_t x, int64_t y) {
  if (__builtin_expect(((x | y) >> 32) == 0, 1)) return (uint32_t)x / (uint32_t)y;
  return x / y;
}
FA_DEVICE int64_t share_begin(int64_t units, int w, int sharers) { return quotient(units * w, sharers); }
// The first unit of the pair after (b, h): false if there is none
template <bool kPrefix = false>
FA_DEVICE bool next_pair(const PagedCache& c, Spot* at) {
  at->unit = 0;
  if (at->h + 1 < c.HK) {
    at->h++;
    return true;
  }
  at->h = 0;
  do at->b++; while (at->b < c.B && units_of<kPrefix>(c, at->b) == 0);
  if (at->b >= c.B) return false;
  at->units = units_of<kPrefix>(c, at->b);
  return true;
}

}  // namespace fa
