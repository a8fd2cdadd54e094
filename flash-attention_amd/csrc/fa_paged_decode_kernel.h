// Attention of a few rows a key head over a paged cache (what is below 32 rows of a product), as a kernel body that fa_paged_decode.hip makes kernels of: over pages in
// 16 bits, and over pages in 8 bits (k8), of whole sequences and of what comes behind a shared prefix (kPrefix).
//
// In 8 bits the values are widened between LDS and the matrix cores.  K: a lane multiplies a key's row, so the row's exponent is the scale of the instruction that
// widens two values, for nothing.  V is read transposed, a lane has one column of eight keys, whose exponents differ: they go into the probabilities instead,
//   o = sum_j (p_j 2^e_j) y_j.
// bf16 has fp32's range: the probability is rounded, and multiplied by a power of two, which rounds nothing.  In fp16, whose e_j lie in -15 .. 8, the largest product has
// to be brought to 1, or the product would lose to fp16's range:
//   p_j 2^e_j = 2^(s_j c + e_j - m'),   m' = max (s_j c + e_j),
// and the sums of the p_j take 2^-e_j back in fp32.  (Not so in bf16: its e_j are up to 220 apart, and of a p_j 2^(e_j - m') that is 0 in fp32 nothing comes back.)
// What is added to the scores is e_j - 1 and not the byte e_j + 127: half a step of fp32 is 2^-18 or 2^-17 at a score with that much too much, up to 5e-6 of the probability
// and of lse.  (The bytes' highest bits are turned for it, 4 instructions for 16 keys: 32 x 12 heads of 10000 keys, d = 32 71.7 -> 72.6 us, d = 64 90.6 -> 91.2, d = 128 as before.)
#pragma once

#include <type_traits>

#include "fa_paged_8bit.h"
#include "fa_paged_line.h"

namespace fa {

// Whether maxima are those of s_j c + e_j, in log2 units, and not of the scores before scaling
template <typename T, bool k8>
constexpr bool kLog2Maxima = k8 && std::is_same_v<T, _Float16>;

// e - 1 of byte i of a word of exponents' bytes (e + 127): that byte with its highest bit turned, as a signed number, which the conversion picks out of the word
FA_DEVICE float exponent_from_one(uint32_t w, int i) { return (float)(int8_t)((w ^ 0x80808080u) >> 8 * i); }

template <int D, int NW_, bool k8>
struct DecodeCfg {
  static constexpr int NW = NW_;
  static constexpr int BN = 32;
  static constexpr int DV = D < 32 ? 32 : D;
  static constexpr int kTile = BN * D * (k8 ? 1 : 2);
  static constexpr int kExps = k8 ? 2 * BN : 0;           // the exponents of a tile's keys, and of its values
  static constexpr int kStage = 2 * kTile + kExps;
  static constexpr int kWave = 2 * kStage;                // two stages of (K tile, V tile)
  static constexpr int kSlack = !k8 && D < 32 ? 64 : 0;   // the 32-wide transposed reads run past a 16-wide V row
  static constexpr int XS = DV + 4;                       // merge: floats per (wave, row)
  static constexpr int kMerge = NW * 32 * XS * 4 + 3 * NW * 32 * 4;
  static constexpr int kTiles = NW * kWave + kSlack;
  static constexpr int kLds = kTiles > kMerge ? kTiles : kMerge;
};

// A pair's part behind a shared prefix: there is one for every pair, of the call's rows (2^24 pairs of 32 rows are counted in 32 bits, for two registers less in scratch)
template <int D>
FA_DEVICE float* whole_part(const PagedFwdParams& p, int b, int h) {
  return p.whole_part + (int64_t)((b * p.c.HK + h) * (p.c.max_sq * p.c.G)) * (D + 4);
}

template <typename T, int D, int NW_, bool k8, bool kPrefix, bool kStream>
FA_DEVICE void paged_decode(const PagedFwdParams p, const int wg, unsigned char* const lds_raw) {
  using C = DecodeCfg<D, NW_, k8>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int NW = C::NW, BN = C::BN, DV = C::DV;
  using KStager = std::conditional_t<k8, GroupStager8<D, kSwzRow, kStream>, GroupStager<D, kSwzRow, kStream>>;
  using VStager = std::conditional_t<k8, GroupStager8<D, kSwzTr, kStream>, GroupStager<D, kSwzTr, kStream>>;
  constexpr int NI = 2 * KStager::NI;  // loads of a tile's K, and of its V
  constexpr int NX = k8 ? 1 : 0;       // ... and of its exponents
  // (Numerator and denominator share the rounding of the probabilities - but not then: a probability times its value's 2^e may be far below fp16's normal numbers while
  // the probability itself is not, and its rounding would be the sum's.)
  constexpr bool kLog2 = kLog2Maxima<T, k8>;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const float cs = p.scale_log2;
  const float mcs = kLog2 ? 1.f : cs;  // what brings a maximum to log2 units

  KStager ks_;
  VStager vs_;
  ks_.init(lane, p.c.k_ss);
  vs_.init(lane, p.c.v_ss);
  unsigned char* const lds_wave = lds_raw + wave * C::kWave;
  // where a lane reads its fragments.  16 bits: elements; 8 bits: bytes, a chunk of 16 for two steps of the product, whose channels are 32 j + 16 hf .. + 15 then
  constexpr int KF = k8 ? (D + 31) / 32 : D / 16;
  int koff[KF], voff[DV / 32];
  if constexpr (k8) {
    const int j16 = lane & 15, key = 4 * hf + ((j16 >> 1) & 3) + 8 * (j16 >> 3), side = (lane >> 4) & 1;
#pragma unroll
    for (int j = 0; j < KF; j++) koff[j] = D == 16 ? c * D + 8 * hf : c * D + 16 * ((2 * j + hf) ^ tile_swz8<D, kSwzRow>(c));
#pragma unroll
    for (int db = 0; db < DV / 32; db++) voff[db] = key * D + (D == 16 ? 0 : 16 * ((2 * db + side) ^ tile_swz8<D, kSwzTr>(key))) + 8 * (j16 & 1);
  } else {
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) koff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);
#pragma unroll
    for (int db = 0; db < DV / 32; db++) voff[db] = tr_off<D, kSwzTr>(0, db * 4, lane);
  }

  // ---- this workgroup's share of the line: [u, u_end), from `at` on
  int64_t u, u_end;
  Spot at;
  if (p.groups > 0) {
    const int sums0 = unit_sums<kPrefix>(p.c, 0);
    const int64_t units = all_units<kPrefix>(p.c, sums0);
    const int n = sharers(p, units);
    if (wg >= n || units == 0) return;
    u = share_begin(units, wg, n);
    u_end = share_begin(units, wg + 1, n);
    at = spot_of<kPrefix>(p.c, u, sums0);
  } else {  // one pair
    const int b = wg / p.c.HK, keys = paged_len(p.c, b) - first_own<kPrefix>(p.c, b);
    at = Spot{b, wg - b * p.c.HK, 0, keys <= kDecodeUnit ? 1 : (keys + kDecodeUnit - 1) / kDecodeUnit};
    u = 0;
    u_end = at.units;
  }

  bool first = true;
  while (u < u_end) {
    const int b = __builtin_amdgcn_readfirstlane(at.b), h = __builtin_amdgcn_readfirstlane(at.h);
    const int unit0 = __builtin_amdgcn_readfirstlane(at.unit), pair_units = __builtin_amdgcn_readfirstlane(at.units);
    const int unit1 = u_end - u < pair_units - unit0 ? unit0 + (int)(u_end - u) : pair_units;
    // a tile's two groups of 16 keys: their pages are asked for a step before they are needed, those of the first two tiles together with the lengths
    // (keys are counted from the sequence's first own one)
    const int first_key = first_own<kPrefix>(p.c, b), skipped = kPrefix ? first_key >> p.c.page_log2 : 0;
    const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs + skipped;
    const int k_lo = unit0 * kDecodeUnit;
    int page[2], page2[2];
    auto ask = [&](int t, int (&to)[2]) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        if constexpr (kPrefix) to[j] = page_of_group(p.c, table, (k_lo >> 4) + 2 * t + j, skipped);
        else to[j] = page_of_group(p.c, table, (k_lo >> 4) + 2 * t + j);
      }
    };
    ask(wave, page);
    ask(wave + NW, page2);
    int q_begin = 0, Lq = 0;
    if (!paged_rows(p.c, b, &q_begin, &Lq)) return;  // (on the line such a sequence has no units)
    const int Lk = own_len<kPrefix>(p.c, b), G = p.c.G, rows = Lq * G;
    const int k_hi = Lk < unit1 * kDecodeUnit ? Lk : unit1 * kDecodeUnit;
    const int ntiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
    const char* const kb = p.c.k + h * p.c.k_hs;
    const char* const vb = p.c.v + h * p.c.v_hs;
    const int last_group = (Lk - 1) >> 4;

    auto issue = [&](int t, int stage, const int (&pages)[2]) {
      unsigned char* const dst = lds_wave + stage * C::kStage;
      const int g0 = (k_lo >> 4) + 2 * t;
      const bool both = g0 < last_group;  // (else the tile's second half repeats the last key, in the first one's page)
      if constexpr (k8) {  // lanes 0 .. 3: the exponents of the first 16 keys, of the others, and the values'
        if (lane < 4) {
          const bool second = both && (lane & 1);
          const int64_t at = ((int64_t)(second ? pages[1] : pages[0]) * p.c.HK + h) << p.c.page_log2;
          dma16_from((lane < 2 ? p.c.k_exps : p.c.v_exps) + at + slot_of_group(p.c, second ? g0 + 1 : g0), dst + 2 * C::kTile);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int g = both ? g0 + j : g0, pg = both ? pages[j] : pages[0];
        ks_.issue(kb + pg * p.c.k_ps + slot_of_group(p.c, g) * p.c.k_ss, p.c.k_ss, g < last_group ? 15 : (Lk - 1) & 15, dst + j * KStager::kBytes);
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int g = both ? g0 + j : g0, pg = both ? pages[j] : pages[0];
        vs_.issue(vb + pg * p.c.v_ps + slot_of_group(p.c, g) * p.c.v_ss, p.c.v_ss, g < last_group ? 15 : (Lk - 1) & 15, dst + C::kTile + j * VStager::kBytes);
      }
    };

    int t = wave, stage = 0;
    if (t < ntiles) issue(t, 0, page);
    if (t + NW < ntiles) issue(t + NW, 1, page2);
    const int row = c < rows ? c : rows - 1;  // (columns past the last row repeat it and are dropped at the end)
    const int tok = row / G;
    vec8 qreg[D / 16];
    {
      const T* qp = reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok) * p.q_rs + (int64_t)(h * G + (row - tok * G)) * p.q_hs + hf * 8;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) qreg[ks] = bitcast<vec8>(ld_global16(qp + (k8 && D > 16 ? (ks >> 1) * 32 + hf * 8 + (ks & 1) * 8 : ks * 16)));
      // waited for here (with the first two tiles): the main loop counts this wave's outstanding loads, these are not to be among them
      wait_vmcnt<0>();
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) asm volatile("" : "+v"(qreg[ks]));
    }
    const int limit = p.causal ? Lk - Lq + tok + 1 : Lk;
    const int least_limit = p.causal ? Lk - Lq + 1 : Lk;  // of row 0

    f32x16 o_acc[DV / 32];
#pragma unroll
    for (int i = 0; i < DV / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) o_acc[i][r] = 0.f;
    float m_i = -INFINITY, l_i = 0.f, u_i = 0.f;  // l_i, u_i: this lane's share, the other half's in lane ^ 32

    for (; t < ntiles; t += NW) {
      const bool next = t + NW < ntiles;  // its 2 * NI loads were issued after this tile's
      if (next) wait_vmcnt<3 * NI + NX>();
      else wait_vmcnt<NI>();
      if (t + 2 * NW < ntiles) ask(t + 2 * NW, page);
      const unsigned char* const tile = lds_wave + stage * C::kStage;
      const T* const Ks = reinterpret_cast<const T*>(lds_wave + stage * C::kStage);
      const T* const Vs = Ks + BN * D;
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = 0.f;
      uint32_t ve[4] = {};  // 8 bits: the exponents of this lane's 16 values
      if constexpr (k8) {
        const unsigned char* const exps = tile + 2 * C::kTile;
        const float scale = power_of_two(exps[c]);
#pragma unroll
        for (int i = 0; i < 4; i++) ve[i] = *reinterpret_cast<const uint32_t*>(exps + BN + 8 * i + 4 * hf);
        if constexpr (D == 16) {
          s = E::mfma32(dequant8<T>(*reinterpret_cast<const u32x2*>(tile + koff[0]), scale), qreg[0], s);
        } else {
#pragma unroll
          for (int j = 0; j < KF; j++) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(tile + koff[j]);
            s = E::mfma32(dequant8<T>(u32x2{w[0], w[1]}, scale), qreg[2 * j], s);
            s = E::mfma32(dequant8<T>(u32x2{w[2], w[3]}, scale), qreg[2 * j + 1], s);
          }
        }
        if constexpr (kLog2) {
#pragma unroll
          for (int r = 0; r < 16; r++) s[r] = __builtin_fmaf(s[r], cs, exponent_from_one(ve[r >> 2], r & 3));
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) s = E::mfma32(*reinterpret_cast<const vec8*>(Ks + koff[ks]), qreg[ks], s);
      }
      const int n0 = k_lo + t * BN;
      if (n0 + BN > least_limit) {
        const int dead = limit - n0 - 4 * hf;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          if (8 * (r >> 2) + (r & 3) < dead) continue;
          s[r] = -INFINITY;
          if constexpr (k8 && !kLog2) ve[r >> 2] &= ~(255u << 8 * (r & 3));  // (behind the sequence's end it may be 255, infinity)
        }
      }
      float mt = s[0];
#pragma unroll
      for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
      mt = half_max(mt);
      if (__any(mt > m_i)) {
        const float m_new = fmaxf(m_i, mt);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2((m_i - m_new) * mcs);
        m_i = m_new;
        l_i *= alpha;
        u_i *= alpha;
#pragma unroll
        for (int i = 0; i < DV / 32; i++) o_acc[i] = o_acc[i] * alpha;
      }
      const float mc = (m_i == -INFINITY ? 0.f : m_i) * mcs;
      vec8 pb[2];
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        f32x8 pf;
        const auto exponent = [&](int i) { return (ve[2 * tt + (i >> 2)] >> 8 * (i & 3)) & 255; };
        if constexpr (kLog2) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            pf[i] = fast_exp2(s[8 * tt + i] - mc);
            u_i = __builtin_fmaf(pf[i], power_of_minus(exponent(i)), u_i);
          }
          pb[tt] = cvt8<T>(pf);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            pf[i] = fast_exp2(__builtin_fmaf(s[8 * tt + i], cs, -mc));
            u_i += pf[i];
          }
          pb[tt] = cvt8<T>(pf);
          l_i = sum8_acc(pb[tt], l_i);
          if constexpr (k8) {
#pragma unroll
            for (int i = 0; i < 8; i++) pf[i] = (float)pb[tt][i] * power_of_two((int)exponent(i));
            pb[tt] = cvt8<T>(pf);
          }
        }
      }
      if (next) wait_vmcnt<2 * NI + NX>();
      else wait_vmcnt<0>();
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
#pragma unroll
        for (int db = 0; db < DV / 32; db++) {
          if constexpr (k8) {
            o_acc[db] = E::mfma32(dequant8<T>(lds_read_tr8(tile + C::kTile + 16 * tt * D + voff[db]), 1.f), pb[tt], o_acc[db]);
          } else {
            const T* vp = Vs + 16 * tt * D + voff[db];
            const u32x2 lo = lds_read_tr16(vp), hi = lds_read_tr16(vp + 8 * D);
            o_acc[db] = E::mfma32(bitcast<vec8>(u32x4{lo[0], lo[1], hi[0], hi[1]}), pb[tt], o_acc[db]);
          }
        }
      if (t + 2 * NW < ntiles) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the stage has been read before it is refilled
        issue(t + 2 * NW, stage, page);
      }
      stage ^= 1;
    }

    // ---- the waves' partial results joined: row r of wave w at X[(w * 32 + r) * XS], m, l and u behind all rows
    __syncthreads();
    float* const X = reinterpret_cast<float*>(lds_raw);
    float* const Xm = X + NW * 32 * C::XS;
    float* const Xl = Xm + NW * 32;
    float* const Xu = Xl + NW * 32;
    l_i = half_sum(l_i);
    u_i = half_sum(u_i);
    if constexpr (kLog2) {
      l_i = u_i;
      m_i += 1.f;  // (from here on results are of 2^m)
    }
    if (c < rows) {
      if (hf == 0) {
        Xm[wave * 32 + c] = m_i;
        Xl[wave * 32 + c] = l_i;
        Xu[wave * 32 + c] = u_i;
      }
#pragma unroll
      for (int db = 0; db < DV / 32; db++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] = o_acc[db][g4 * 4 + i];
          *reinterpret_cast<f32x4*>(X + (wave * 32 + c) * C::XS + db * 32 + g4 * 8 + hf * 4) = x;
        }
    }
    __syncthreads();
    // (behind a prefix a whole pair's results are a part, too: the join adds the prefix's)
    const bool alone = unit0 == 0 && unit1 == pair_units, whole = alone && !kPrefix;
    float* const part = whole ? nullptr : kPrefix && alone ? whole_part<D>(p, b, h) : p.part + ((int64_t)wg * 2 + (first ? 0 : 1)) * (kPartRows * (D + 4));
    for (int idx = tid; idx < rows * (D / 4); idx += 64 * NW) {
      const int r = idx / (D / 4), d0 = idx % (D / 4) * 4;
      float m = Xm[r];
#pragma unroll
      for (int w = 1; w < NW; w++) m = fmaxf(m, Xm[w * 32 + r]);
      const float mu = m == -INFINITY ? 0.f : m;
      float l = 0.f, us = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float f = fast_exp2((Xm[w * 32 + r] - mu) * mcs);  // 0 for a wave without keys
        l = __builtin_fmaf(Xl[w * 32 + r], f, l);
        us = __builtin_fmaf(Xu[w * 32 + r], f, us);
        o = o + *reinterpret_cast<const f32x4*>(X + (w * 32 + r) * C::XS + d0) * f;
      }
      if (whole) {
        store_row_piece<T>(p, q_begin, h, r, d0, o * (l > 0.f ? fast_rcp(l) : 1.f));
        if (d0 == 0) store_lse(p, b, h, r, lse_of(m, us, mcs));
      } else {
        *reinterpret_cast<f32x4*>(part + r * (D + 4) + d0) = o;
        if (d0 == 0) {
          float* const ml = part + r * (D + 4) + D;
          ml[0] = m;
          ml[1] = l;
          ml[2] = us;
        }
      }
    }
    first = false;
    u += unit1 - unit0;
    if (u >= u_end) return;
    if (!next_pair<kPrefix>(p.c, &at)) return;  // (never: the line does not end here)
    __syncthreads();  // the joined results have been read before the tiles come in over them
  }
}

// The pairs that the ends of the workgroups' shares have cut (blockIdx.x: a pair; blockIdx.y and the threads share its rows): D / 4 threads over a row's
// elements, times lanes over its parts - as many as there are, rounded up to a power of two -, times rows side by side.  The lanes' results are
// joined in LDS, in the same order each time.
template <typename T, int D, bool k8, bool kPrefix>
FA_DEVICE void paged_decode_join(const PagedFwdParams p) {
  constexpr int kCols = D / 4, kLanes = 256 / kCols;
  __shared__ f32x4 os[256];
  __shared__ PartRow ms[256];
  const int b = blockIdx.x / p.c.HK, h = (int)blockIdx.x - b * p.c.HK;
  int64_t units = 0, begin = 0;  // of all pairs; where this one's lie
  int pair_units = 0;
  for (int first = 0; first < p.c.B; first += 64) {
    const int sums = unit_sums<kPrefix>(p.c, first), k = b - first;
    if (k >= 0 && k < 64) {
      const int upto = k > 0 ? __builtin_amdgcn_readlane(sums, k > 0 ? k - 1 : 0) : 0;
      pair_units = __builtin_amdgcn_readlane(sums, k) - upto;
      begin = (units + upto) * p.c.HK + (int64_t)h * pair_units;
    }
    units += __builtin_amdgcn_readlane(sums, 63);
  }
  units *= p.c.HK;
  int q_begin = 0, Lq = 0;
  if (pair_units == 0 || !paged_rows(p.c, b, &q_begin, &Lq)) return;
  const int n = sharers(p, units);
  const auto share_of = [&](int64_t u) { return (int)quotient((u + 1) * n - 1, units); };  // (the last w with units * w / n <= u)
  const int w0 = share_of(begin), w1 = share_of(begin + pair_units - 1);
  const bool alone = w0 == w1;
  if (alone && !kPrefix) return;
  constexpr bool kLog2 = kLog2Maxima<T, k8>;
  const float cs = kLog2 ? 1.f : p.scale_log2;
  // the pair is the last of share w0, and its first, too, if the share begins with it; it is the first of the others'
  const int first_slot = share_begin(units, w0, n) == begin ? 0 : 1;
  const bool shares = kPrefix && first_own<kPrefix>(p.c, b) > 0;
  const int parts = w1 - w0 + 1 + (shares ? p.pre_splits : 0);
  // (behind prefixes more than 1024 rows: eight parts a lane, since what the lanes do for each other fills the device then.  us with one / eight: 64 sequences of 8 x 4
  // heads behind 16384 keys 62.4 / 61.2, behind 32768 74.6 / 73.1; 12 of 4 x 3 heads, 3 tokens, 16.8 / 17.2; 32 of 8 x 4 heads 32.3 / 32.3)
  const int each = kPrefix && (int64_t)gridDim.x * (p.c.max_sq * p.c.G) > 1024 ? 8 : 1;
  int lanes = 2;
  while (lanes < kLanes && lanes * each < parts) lanes *= 2;
  const int col = threadIdx.x % kCols, at = threadIdx.x / kCols, lane = at & (lanes - 1), side = at / lanes, beside = kLanes / lanes;
  const int rows = Lq * p.c.G;
  for (int r0 = blockIdx.y * beside; r0 < rows; r0 += gridDim.y * beside) {
    const int r = r0 + side;
    JoinedRow x;
    if (r < rows) {
      if (shares) add_prefix<D>(p, &x, h, (int64_t)q_begin * p.c.G + r, col * 4, cs, kLog2 ? p.scale_log2 : 1.f, lane, lanes);
      // (several parts' loads on their way together: us, then, and else: 1 pair of 100000 keys, d = 128 24.2 / 35.4, in 8 bits 23.9 / 38.8, of 30000 15.8 / 22.3; 8 of 8000
      // 14.6 / 15.4; 16 of 7000, d = 64 13.35 / 13.25)
#pragma unroll 4
      for (int i = w0 + lane; i <= w1; i += lanes) {
        const float* const s = (kPrefix && alone ? whole_part<D>(p, b, h) : p.part + ((int64_t)i * 2 + (i == w0 ? first_slot : 0)) * (kPartRows * (D + 4))) + r * (D + 4);
        x.add(PartRow{s[D], s[D + 1], s[D + 2]}, *reinterpret_cast<const f32x4*>(s + col * 4), cs);
      }
    }
    x.across<kCols>(lane, lanes, cs, os, ms);
    if (lane == 0 && r < rows) {
      store_row_piece<T>(p, q_begin, h, r, col * 4, x.o * (x.a.l > 0.f ? fast_rcp(x.a.l) : 1.f));
      if (col == 0) store_lse(p, b, h, r, lse_of(x.a.m, x.a.u, cs));
    }
  }
}

// A workgroup a pair, and others beside it for its rows
inline hipError_t launch_decode_join(void (*join)(PagedFwdParams), const PagedFwdParams& p, hipStream_t stream) {
  const unsigned pairs = (unsigned)(p.c.B * p.c.HK), rows = (unsigned)(p.c.max_sq * p.c.G), side = pairs < 1024 ? 1024 / pairs : 1;
  hipLaunchKernelGGL(join, dim3(pairs, rows < side ? rows : side), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// A decode kernel's launch, and behind it, where workgroups share the line, the join
inline hipError_t launch_decode(void (*kernel)(PagedFwdParams), int waves, void (*join)(PagedFwdParams), const PagedFwdParams& p, hipStream_t stream) {
  const unsigned pairs = (unsigned)(p.c.B * p.c.HK);
  hipLaunchKernelGGL(kernel, dim3(p.groups > 0 ? (unsigned)p.groups : pairs), dim3(64 * waves), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.groups == 0 ? e : launch_decode_join(join, p, stream);
}

}  // namespace fa
