// Attention of many rows a key head over a paged cache, as a kernel body that fa_paged_chunk.hip, fa_paged_chunk_8bit.hip and fa_paged_prefix_kernel.h make kernels of: over
// pages in 16 bits, whose tiles go from memory to LDS by themselves, and in 8 bits (k8), whose tiles are widened on the way: a thread holds the next tile's chunks (16 values
// each) in registers while the waves compute, and writes what they stand for, in 16 bits, into the buffer that nobody reads; each value is widened once for the workgroup's 128
// rows, and the main loop is the same.  kShared: the rows of a group of sequences over the keys that the group shares, without a mask; partial results.
#pragma once

#include <type_traits>

#include "fa_paged_8bit.h"
#include "fa_paged_fwd.h"

namespace fa {

constexpr int chunk_keys(int head_dim) { return head_dim == 128 ? 32 : 64; }  // keys of a tile
template <int D, int BN_ = chunk_keys(D)>
struct ChunkCfg {
  static constexpr int BN = BN_;
  static constexpr int DV = D < 32 ? 32 : D;
  static constexpr int kTile = BN * D * 2;
  static constexpr int kBuf = 2 * kTile;
  static constexpr int kSlack = D < 32 ? 64 : 0;
  static constexpr int OS = D + 8;  // stride of the output's way through LDS
  static constexpr int kOut = 128 * OS * 2;
  static constexpr int kLds = 2 * kBuf + kSlack > kOut ? 2 * kBuf + kSlack : kOut;
  // Waves per SIMD; with the second sum that lse wants one less, without registers in scratch (d = 64: 44 of them).  Without lse d = 128 keeps the third
  // wave and eight registers in scratch: 16 x 1024 tokens of 32 heads behind 5120 keys 1427 us (1060 TFLOP/s), with two waves 1550.
  static constexpr int kWaves = D == 128 ? 3 : 4;
};

// The sequence with the rank-th largest number of keys (ties: lower index first); more than 64: in their order.
FA_DEVICE int longest_sequence(const PagedCache& c, int rank) {
  if (c.B > 64 || c.B < 2) return rank;
  const int lane = threadIdx.x & 63;
  const int len = keys_in_reach(c.seqlens[lane < c.B ? lane : c.B - 1], c.max_keys);
  int before = 0;
  for (int j = 0; j < c.B; j++) {
    const int lj = __builtin_amdgcn_readlane(len, j);
    before += (lj > len || (lj == len && j < lane)) ? 1 : 0;
  }
  const uint64_t hit = __builtin_amdgcn_ballot_w64(lane < c.B && before == rank);
  return __builtin_amdgcn_readfirstlane(hit != 0 ? (int)__builtin_ctzll(hit) : rank);
}

// Workgroup id -> (sequence, key head, row tile).  Ids go to the eight XCDs in turn; the tiles of a pair should run on one of them, side by side, since
// they read the same keys, and the longest sequences should begin first.  With pairs enough (p.deal) those are dealt to the XCDs one by one, longest
// sequences first: 4 sequences of 4096 .. 8192 keys, 8 key heads, 1024 new tokens each, d = 128 421 us (to 429 on other boxes), in contiguous pieces, which give an XCD
// one sequence's heads, 516.  Few pairs: each XCD takes a contiguous piece of the line of all tiles.  Tiles of a pair from the last (longest walk under the mask) on.
FA_DEVICE bool place(const PagedFwdParams& p, int id, int* b, int* h, int* tile) {
  const int pairs = p.c.B * p.c.HK, x = id & 7, j = id >> 3;
  int64_t at;
  if (p.deal) {
    const int64_t rank = x + 8 * (int64_t)(j / p.nq_tiles);
    if (rank >= pairs) return false;
    at = rank * p.nq_tiles + j % p.nq_tiles;
  } else {
    const int64_t items = (int64_t)pairs * p.nq_tiles, each = (items + 7) / 8;
    at = x * each + j;
    if (j >= each || at >= items) return false;
  }
  const int rank = (int)(at / p.nq_tiles);
  *tile = p.nq_tiles - 1 - (int)(at - (int64_t)rank * p.nq_tiles);
  const int s = rank / p.c.HK;
  *h = rank - s * p.c.HK;
  *b = longest_sequence(p.c, s);
  return true;
}

// Workgroup id -> (group, key head, row tile) of a launch over shared prefixes: tiles of all groups in one line, g by g.  The tiles of a key head read the same keys of a
// group: each XCD takes a contiguous piece of (head, tile).
FA_DEVICE bool place_shared(const PagedFwdParams& p, int id, int* g, int* h, int* tile) {
  const int64_t items = (int64_t)p.c.HK * p.pre_tiles, each = (items + 7) / 8, at = (id & 7) * each + (id >> 3);
  if ((id >> 3) >= each || at >= items) return false;
  *h = (int)(at / p.pre_tiles);
  int rest = (int)(at - (int64_t)*h * p.pre_tiles);
  if (p.n_groups == 1) {
    *g = 0;
    *tile = rest;
    return true;
  }
  for (int first = 0; first < p.n_groups; first += 64) {
    const int i = first + (threadIdx.x & 63);
    int q0 = 0, tokens = 0, b0 = 0;
    if (i < p.n_groups && group_rows(p, i, &b0, &q0, &tokens)) tokens = (tokens * p.c.G + kChunkRows - 1) / kChunkRows;
    const int sums = wave_prefix_sum(tokens), all = __builtin_amdgcn_readlane(sums, 63);
    if (rest < all) {
      const int lane = __popcll(__ballot(sums <= rest));
      *g = first + lane;
      *tile = rest - (lane > 0 ? __builtin_amdgcn_readlane(sums, lane > 0 ? lane - 1 : 0) : 0);
      return true;
    }
    rest -= all;
  }
  return false;
}

template <typename T, int D, bool kLse, bool k8, bool kShared, int BN_ = chunk_keys(D)>
FA_DEVICE void paged_chunk(const PagedFwdParams p, const int wg, const int split, unsigned char* const lds_raw) {
  using C = ChunkCfg<D, BN_>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int BN = C::BN, DV = C::DV, KB = BN / 32, CH = D / 8;
  constexpr int GW = BN / 32;  // groups of 16 keys that a wave stages (waves 0 and 1: K, 2 and 3: V)

  int b, h, qt;
  int q_begin = 0, Lq = 0, Lk = 0;
  if constexpr (kShared) {
    int g = 0;
    if (!place_shared(p, wg, &g, &h, &qt)) return;
    if (!group_rows(p, __builtin_amdgcn_readfirstlane(g), &b, &q_begin, &Lq)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    q_begin = __builtin_amdgcn_readfirstlane(q_begin);
    Lq = __builtin_amdgcn_readfirstlane(Lq);
    Lk = first_own<true>(p.c, b);
    if (Lk == 0) return;  // (nothing is shared, nobody looks for a part)
  } else {
    if (!place(p, wg, &b, &h, &qt)) return;
    if (!paged_rows(p.c, b, &q_begin, &Lq)) return;
  }
  const int G = p.c.G, rows = Lq * G, m0 = qt * kChunkRows;
  if (m0 >= rows) return;
  if constexpr (!kShared) Lk = paged_len(p.c, b);
  const bool masked = !kShared && p.causal;
  const int n_splits = kShared ? p.pre_splits : p.n_splits;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const int mw = m0 + wave * 32;
  const bool wave_live = mw < rows;
  const int row = mw + c < rows ? mw + c : rows - 1;  // (rows past the end repeat the last one and are not stored)
  const int tok = row / G;

  vec8 qreg[D / 16];
  {
    const T* qp = reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok) * p.q_rs + (int64_t)(h * G + (row - tok * G)) * p.q_hs + hf * 8;
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) qreg[ks] = bitcast<vec8>(ld_global16(qp + ks * 16));
  }
  // keys that this lane's row, the wave's first row and the workgroup's last row see
  const int past = Lk - Lq + 1;
  const int limit = masked ? past + tok : Lk;
  const int first_row = mw < rows ? mw : rows - 1, last_row = m0 + kChunkRows < rows ? m0 + kChunkRows - 1 : rows - 1;
  const int last_in_wave = mw + 31 < rows ? mw + 31 : rows - 1;
  const int least_limit = __builtin_amdgcn_readfirstlane(masked ? past + first_row / G : Lk);
  const int wave_limit = __builtin_amdgcn_readfirstlane(masked ? past + last_in_wave / G : Lk);
  int n_end = masked ? past + last_row / G : Lk;
  n_end = n_end > 0 ? n_end : 0;
  const int ntiles_all = (n_end + BN - 1) / BN;
  const int tile0 = (int)((int64_t)split * ntiles_all / n_splits);
  const int ntiles = (int)((int64_t)(split + 1) * ntiles_all / n_splits);

  // ---- staging
  const bool stages_v = wave >= 2;
  const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
  const int last_group = (Lk - 1) >> 4;
  // (a prefix is read by a row tile or two, and past the caches: 32 sequences of 8 x 4 heads behind 32768 keys 45.8 -> 43.2 us, 64, two tiles, behind 8192 35.3 -> 34.7; in 8
  // bits, through registers, it makes no difference)
  GroupStager<D, kSwzRow, kShared> sk;
  GroupStager<D, kSwzTr, kShared> sv;
  if constexpr (!k8) {
    if (stages_v) sv.init(lane, p.c.v_ss);
    else sk.init(lane, p.c.k_ss);
  }
  const char* const base = stages_v ? p.c.v + h * p.c.v_hs : p.c.k + h * p.c.k_hs;
  const int64_t page_stride = stages_v ? p.c.v_ps : p.c.k_ps, slot_stride = stages_v ? p.c.v_ss : p.c.k_ss;
  const int group0 = (wave & 1) * GW;
  int page[GW];
  auto ask = [&](int it) {
#pragma unroll
    for (int j = 0; j < GW; j++) {
      const int g = it * (BN / 16) + group0 + j;
      page[j] = page_of_group(p.c, table, g < last_group ? g : last_group);
    }
  };
  auto stage = [&](int it, int buf) {
    unsigned char* const dst = lds_raw + buf * C::kBuf + (stages_v ? C::kTile : 0) + group0 * GroupStager<D, kSwzRow>::kBytes;
#pragma unroll
    for (int j = 0; j < GW; j++) {
      const int g0 = it * (BN / 16) + group0 + j, g = g0 < last_group ? g0 : last_group;
      const char* const from = base + page[j] * page_stride + slot_of_group(p.c, g) * slot_stride;
      const int last = g < last_group ? 15 : (Lk - 1) & 15;
      if (stages_v) sv.issue(from, slot_stride, last, dst + j * GroupStager<D, kSwzRow>::kBytes);
      else sk.issue(from, slot_stride, last, dst + j * GroupStager<D, kSwzRow>::kBytes);
    }
  };

  // ---- staging of pages in 8 bits: this thread's chunks of a tile (d >= 64: one of K and one of V; d < 64: one of either).  A wave's rows lie in one or, at d < 64, several
  // groups of 16 keys, a page each: for one group addresses are a wave-uniform base and the lane's offset.
  constexpr int kChunks = BN * D / 16, CH8 = D / 16, kSets = kChunks > 256 ? kChunks / 256 : 1, kMine = kChunks >= 256 ? 2 : 1;
  constexpr int kWaveRows = 64 / CH8, kGroups = kWaveRows > 16 ? kWaveRows / 16 : 1, kSetRows = kChunks / kSets / CH8;
  const int my = tid % (kChunks / kSets), my_row = my / CH8, my_chunk = my % CH8;  // (of the first set; the others' rows are kSetRows further)
  const bool mine = kMine == 2 || tid < 2 * kChunks, my_v = kMine == 1 && tid >= kChunks;
  const int wave_row = (wave * 64) % (kChunks / kSets) / CH8;  // (kMine == 1: a wave is K's or V's)
  const uint32_t k_off = (uint32_t)((my_row & 15) * p.c.k_ss) + 16u * my_chunk, v_off = (uint32_t)((my_row & 15) * p.c.v_ss) + 16u * my_chunk;
  u32x4 raw[kSets][kMine];
  int raw_exp[kSets][kMine], page8[kSets][kGroups];
  auto ask8 = [&](int it) {  // the pages of the wave's rows of tile `it`, a step before they are needed
#pragma unroll
    for (int i = 0; i < kSets; i++)
#pragma unroll
      for (int j = 0; j < kGroups; j++) {
        const int g = (it * BN + i * kSetRows + wave_row) / 16 + j;
        page8[i][j] = page_of_group(p.c, table, g < last_group ? g : last_group);
      }
  };
  auto fetch = [&](int it) {
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < kSets; i++) {
      const int n0 = it * BN + i * kSetRows, g0 = (n0 + wave_row) / 16;
      int64_t page = page8[i][0];
      int g = g0 < last_group ? g0 : last_group;
      if constexpr (kGroups > 1) {
        const int in = (my_row >> 4) & (kGroups - 1);
#pragma unroll
        for (int j = 1; j < kGroups; j++)
          if (in == j) page = page8[i][j];
        g = g0 + in < last_group ? g0 + in : last_group;
      }
      const int slot = slot_of_group(p.c, g);
      const char* const kb = p.c.k + h * p.c.k_hs + page * p.c.k_ps + slot * p.c.k_ss;
      const char* const vb = p.c.v + h * p.c.v_hs + page * p.c.v_ps + slot * p.c.v_ss;
      const int64_t xb = ((page * p.c.HK + h) << p.c.page_log2) + slot;
      uint32_t ko = k_off, vo = v_off, row = my_row & 15;
      if (__builtin_expect(n0 + kSetRows > Lk, 0)) {  // (rows behind the last key repeat it)
        const int last = (Lk - 1) & 15;
        if (n0 + my_row >= Lk) {
          row = last;
          ko = (uint32_t)(last * p.c.k_ss) + 16u * my_chunk;
          vo = (uint32_t)(last * p.c.v_ss) + 16u * my_chunk;
        }
      }
      if constexpr (kMine == 2) {
        raw[i][0] = ld_global16(kb + ko);
        raw_exp[i][0] = p.c.k_exps[xb + row];
        raw[i][1] = ld_global16(vb + vo);
        raw_exp[i][1] = p.c.v_exps[xb + row];
      } else {
        raw[i][0] = ld_global16(my_v ? vb + vo : kb + ko);
        raw_exp[i][0] = (my_v ? p.c.v_exps : p.c.k_exps)[xb + row];
      }
    }
  };
  auto widen = [&](int buf) {
    if (!mine) return;
    T* const to = reinterpret_cast<T*>(lds_raw + buf * C::kBuf);
#pragma unroll
    for (int i = 0; i < kSets; i++)
#pragma unroll
      for (int m = 0; m < kMine; m++) {
        const float scale = power_of_two(raw_exp[i][m]);
        const bool is_v = m == 1 || my_v;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int row = i * kSetRows + my_row, chunk = 2 * my_chunk + j;
          *reinterpret_cast<vec8*>(to + (is_v ? BN * D + frag_off<D, kSwzTr>(row, chunk) : frag_off<D, kSwzRow>(row, chunk))) =
              dequant8<T>(u32x2{raw[i][m][2 * j], raw[i][m][2 * j + 1]}, scale);
        }
      }
  };

  f32x16 o_acc[DV / 32];
#pragma unroll
  for (int i = 0; i < DV / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) o_acc[i][r] = 0.f;
  float m_i = -INFINITY, l_i = 0.f, u_i = 0.f;
  const float cs = p.scale_log2;
  int voff[DV / 32], koff[D / 16];
#pragma unroll
  for (int db = 0; db < DV / 32; db++) voff[db] = tr_off<D, kSwzTr>(0, db * 4, lane);
#pragma unroll
  for (int ks = 0; ks < D / 16; ks++) koff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);

  int buf = 0, it = tile0;
  if (it < ntiles) {
    if constexpr (k8) {
      ask8(it);
      fetch(it);
      if (it + 1 < ntiles) ask8(it + 1);
      widen(0);
      if (it + 1 < ntiles) fetch(it + 1);
      if (it + 2 < ntiles) ask8(it + 2);
    } else {
      ask(it);
      stage(it, 0);
      if (it + 1 < ntiles) ask(it + 1);
    }
  }
  asm volatile(".p2align 7");
  while (it < ntiles) {
    const int n0 = it * BN;
#pragma unroll
    for (int i = 0; i < DV / 32; i++) asm volatile("" : "+v"(o_acc[i]));  // (see fa_fwd_kernel.h: keeps O from being copied on every trip)
    if constexpr (k8) {
      __syncthreads();  // tile `it` is in LDS, and nobody still reads the other buffer
    } else {
      wait_vmem();      // this wave's share of tile `it` is in LDS
      __syncthreads();  // so is everyone else's, and nobody still reads the other buffer
      if (it + 1 < ntiles) {
        stage(it + 1, buf ^ 1);
        if (it + 2 < ntiles) ask(it + 2);
      }
    }
    const T* const Ks = reinterpret_cast<const T*>(lds_raw + buf * C::kBuf);
    const T* const Vs = Ks + BN * D;
    buf ^= 1;

    if (wave_live && n0 < wave_limit) {
      f32x16 s[KB];
      auto scores = [&]() {
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
#pragma unroll
          for (int r = 0; r < 16; r++) s[kb][r] = 0.f;
#pragma unroll
          for (int ks = 0; ks < D / 16; ks++) s[kb] = E::mfma32(*reinterpret_cast<const vec8*>(Ks + kb * 32 * D + koff[ks]), qreg[ks], s[kb]);
        }
        if (n0 + BN > least_limit) {
          int dead = limit - n0 - 4 * hf;
          asm volatile("" : "+v"(dead));
#pragma unroll
          for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
              if (kb * 32 + (r >> 2) * 8 + (r & 3) >= dead) s[kb][r] = -INFINITY;
              if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);
            }
        }
      };
      vec8 pb[KB][2];
      float lt, ut;
      auto probabilities = [&]() {
        const float mc = (m_i == -INFINITY ? 0.f : m_i) * cs;
        lt = 0.f;
        ut = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            s[kb][r] = fast_exp2(__builtin_fmaf(s[kb][r], cs, -mc));
            if (kLse) ut += s[kb][r];
          }
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
          for (int t = 0; t < 2; t++) {
            f32x8 pf;
#pragma unroll
            for (int i = 0; i < 8; i++) pf[i] = s[kb][8 * t + i];
            pb[kb][t] = cvt8<T>(pf);
            lt = sum8_acc(pb[kb][t], lt);
            if constexpr (D <= 64) asm volatile("" : "+v"(pb[kb][t]));
          }
      };
      // (the reference point of the exponentials moves only when a lane's row sum says that it has to: see fa_fwd_kernel.h)
      scores();
      bool redo = __any(m_i == -INFINITY);
      if (!redo) {
        probabilities();
        redo = __any(!(lt <= kRescaleLimit));  // (inf and NaN, too)
        if (__builtin_expect(redo, 0)) scores();
      }
      if (__builtin_expect(redo, 0)) {
        float mt = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
          for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[kb][r]);
        mt = half_max(mt);
        const float m_new = fmaxf(m_i, mt);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(m_i * cs - m_use * cs);
        m_i = m_new;
        l_i *= alpha;
        u_i *= alpha;
#pragma unroll
        for (int i = 0; i < DV / 32; i++) o_acc[i] = o_acc[i] * alpha;
        probabilities();
      }
      l_i += lt;
      u_i += ut;
#pragma unroll
      for (int kb = 0; kb < KB; kb++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int db = 0; db < DV / 32; db++) {
            const T* vp = Vs + (kb * 32 + 16 * t) * D + voff[db];
            const u32x2 lo = lds_read_tr16(vp), hi = lds_read_tr16(vp + 8 * D);
            o_acc[db] = E::mfma32(bitcast<vec8>(u32x4{lo[0], lo[1], hi[0], hi[1]}), pb[kb][t], o_acc[db]);
          }
    }
    if constexpr (k8) {  // (in front of the products the next tile's writes cost 451 us where they cost 431 here: 4 x 1024 tokens over 4096 .. 8192 keys, 8 heads of 32)
      if (it + 1 < ntiles) widen(buf);
      if (it + 2 < ntiles) fetch(it + 2);
      if (it + 3 < ntiles) ask8(it + 3);
    }
    it++;
  }

  const float l_tot = half_sum(l_i);
  const float u_tot = kLse ? half_sum(u_i) : 0.f;
  if (kShared || n_splits > 1) {  // partial result of this split, fp32: [split][pair][row of nq_tiles * 128][D], m, l and u behind all of them
    if (mw + c < rows) {
      // (of a prefix: [split][key head][row of the call])
      const int64_t part_rows = kShared ? prefix_part_rows(p.c.total_q, G) : (int64_t)p.nq_tiles * kChunkRows;
      const int64_t all = (kShared ? p.c.HK : (int64_t)p.c.B * p.c.HK) * part_rows;
      const int64_t at = kShared ? h * part_rows + (int64_t)q_begin * G + mw + c : ((int64_t)b * p.c.HK + h) * part_rows + mw + c;
      float* const parts = kShared ? p.pre : p.part;
      float* const op = parts + (int64_t)split * all * (D + 3) + at * D;
      if (hf == 0) {
        float* const ml = parts + (int64_t)split * all * (D + 3) + all * D + at * 3;
        ml[0] = m_i;
        ml[1] = l_tot;
        ml[2] = u_tot;
      }
#pragma unroll
      for (int db = 0; db < DV / 32; db++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
          const int d0 = db * 32 + g4 * 8 + hf * 4;
          if (d0 < D) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = o_acc[db][g4 * 4 + i];
            *reinterpret_cast<f32x4*>(op + d0) = x;
          }
        }
    }
    return;
  }
  const float inv = l_tot > 0.f ? fast_rcp(l_tot) : 1.f;
  if (kLse && hf == 0 && mw + c < rows) store_lse(p, b, h, mw + c, lse_of(m_i, u_tot, cs));
  __syncthreads();  // every wave has left the tiles
  T* const Os = reinterpret_cast<T*>(lds_raw) + wave * 32 * C::OS;
#pragma unroll
  for (int db = 0; db < DV / 32; db++)
#pragma unroll
    for (int g4 = 0; g4 < 4; g4++) {
      const int d0 = db * 32 + g4 * 8 + hf * 4;
      if (d0 < D) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = o_acc[db][g4 * 4 + i] * inv;
        *reinterpret_cast<typename E::vec4*>(Os + c * C::OS + d0) = cvt4<T>(x);
      }
    }
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's LDS writes have landed
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < (32 * CH + 63) / 64; i++) {
    const int ch = lane + i * 64, r = ch / CH, col = (ch % CH) * 8;
    if ((32 * CH % 64 == 0 || ch < 32 * CH) && mw + r < rows) {
      const int t = (mw + r) / G, g = mw + r - t * G;
      st_global16(reinterpret_cast<T*>(p.o) + (int64_t)(q_begin + t) * p.o_rs + (int64_t)(h * G + g) * p.o_hs + col,
                  *reinterpret_cast<const u32x4*>(Os + r * C::OS + col));
    }
  }
}

// Threads of a row's elements times lanes over its splits, four of them each where there are lanes enough (62 splits of 64 rows, 8 key heads, d = 128
// 7 us, with one lane 34).
template <int D>
constexpr int kJoinCols = D / 4;
template <int D>
int join_lanes(int n_splits) {
  int lanes = 1;
  while (lanes < 256 / kJoinCols<D> && lanes * 4 < n_splits) lanes *= 2;
  return lanes;
}
// The splits' partial results joined.
template <typename T, int D>
FA_DEVICE void paged_chunk_join(const PagedFwdParams p, int lanes) {
  constexpr int kCols = kJoinCols<D>;
  __shared__ f32x4 os[256];
  __shared__ PartRow ms[256];
  const int64_t all = (int64_t)p.c.B * p.c.HK * p.nq_tiles * kChunkRows;
  const int col = threadIdx.x % kCols, in = threadIdx.x / kCols, lane = in & (lanes - 1);
  const int64_t at = (int64_t)blockIdx.x * (256 / kCols / lanes) + in / lanes;
  const int pair = (int)(at / (p.nq_tiles * kChunkRows)), r = (int)(at - (int64_t)pair * p.nq_tiles * kChunkRows);
  const int b = pair / p.c.HK, h = pair - b * p.c.HK;
  int s = 0, e = 0;
  if (at < all) {
    s = p.c.cu_q[b];
    e = p.c.cu_q[b + 1];
  }
  const bool on = s >= 0 && e > s && e <= p.c.total_q && r < (e - s < p.c.max_sq ? e - s : p.c.max_sq) * p.c.G;
  const float cs = p.scale_log2;
  JoinedRow x;
  if (on) {
#pragma unroll 4
    for (int i = lane; i < p.n_splits; i += lanes) {
      const float* const from = p.part + (int64_t)i * all * (D + 3);
      const float* const ml = from + all * D + at * 3;
      x.add(PartRow{ml[0], ml[1], ml[2]}, *reinterpret_cast<const f32x4*>(from + at * D + col * 4), cs);
    }
  }
  x.across<kCols>(lane, lanes, cs, os, ms);
  if (on && lane == 0) {
    store_row_piece<T>(p, s, h, r, col * 4, x.o * (x.a.l > 0.f ? fast_rcp(x.a.l) : 1.f));
    if (col == 0) store_lse(p, b, h, r, lse_of(x.a.m, x.a.u, cs));
  }
}

// A chunk kernel's launch, and behind it, where row tiles share their keys, the join
inline hipError_t launch_chunk(void (*kernel)(PagedFwdParams), const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  const int64_t pairs = (int64_t)p.c.B * p.c.HK, items = pairs * p.nq_tiles;
  const dim3 grid((unsigned)(p.deal ? (pairs + 7) / 8 * 8 * p.nq_tiles : (items + 7) / 8 * 8), (unsigned)p.n_splits);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.n_splits <= 1 ? e : launch_paged_chunk_join(p, dtype, head_dim, stream);
}

}  // namespace fa
