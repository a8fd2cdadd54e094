// Attention of a chunk of new tokens over a paged cache: G * Lq rows a key head, any number of them.
//
// The forward kernel's plan (fa_fwd_kernel.h): a workgroup of four waves owns 128 rows, 32 a wave, and streams tiles of K and V through a double
// buffer in LDS; S^T = K Q^T and O^T = V^T P^T keep a row in a lane, its maximum moves only where it has to.  What differs: a tile's rows come from pages, in
// groups of 16 that lie in one page each (their addresses are made by scalar instructions, their pages asked for a step ahead through the scalar cache),
// rows are heads of a group times tokens, so that a key head's keys are read once per 128 of them, and the causal mask is aligned at the end.
// Bound by the matrix cores and the exponentials; launches of few rows and many keys share a row tile's keys among workgroups (n_splits) and
// join their partial results in a second kernel.
#include "fa_paged_fwd.h"

namespace fa {

namespace {

template <int D>
struct ChunkCfg {
  static constexpr int BN = D == 128 ? 32 : 64;
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

}  // namespace

template <typename T, int D, bool kLse>
__global__ void __launch_bounds__(256, ChunkCfg<D>::kWaves - (kLse ? 1 : 0)) fa_paged_chunk_kernel(const PagedFwdParams p) {
  using C = ChunkCfg<D>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int BN = C::BN, DV = C::DV, KB = BN / 32, CH = D / 8;
  constexpr int GW = BN / 32;  // groups of 16 keys that a wave stages (waves 0 and 1: K, 2 and 3: V)
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[C::kLds];

  int b, h, qt;
  if (!place(p, blockIdx.x, &b, &h, &qt)) return;
  const int split = blockIdx.y;
  int q_begin = 0, Lq = 0;
  if (!paged_rows(p.c, b, &q_begin, &Lq)) return;
  const int G = p.c.G, rows = Lq * G, m0 = qt * kChunkRows;
  if (m0 >= rows) return;
  const int Lk = paged_len(p.c, b);

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
  const int limit = p.causal ? past + tok : Lk;
  const int first_row = mw < rows ? mw : rows - 1, last_row = m0 + kChunkRows < rows ? m0 + kChunkRows - 1 : rows - 1;
  const int last_in_wave = mw + 31 < rows ? mw + 31 : rows - 1;
  const int least_limit = __builtin_amdgcn_readfirstlane(p.causal ? past + first_row / G : Lk);
  const int wave_limit = __builtin_amdgcn_readfirstlane(p.causal ? past + last_in_wave / G : Lk);
  int n_end = p.causal ? past + last_row / G : Lk;
  n_end = n_end > 0 ? n_end : 0;
  const int ntiles_all = (n_end + BN - 1) / BN;
  const int tile0 = (int)((int64_t)split * ntiles_all / p.n_splits);
  const int ntiles = (int)((int64_t)(split + 1) * ntiles_all / p.n_splits);

  // ---- staging
  const bool stages_v = wave >= 2;
  const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
  const int last_group = (Lk - 1) >> 4;
  GroupStager<D, kSwzRow> sk;
  GroupStager<D, kSwzTr> sv;
  if (stages_v) sv.init(lane, p.c.v_ss);
  else sk.init(lane, p.c.k_ss);
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
    ask(it);
    stage(it, 0);
    if (it + 1 < ntiles) ask(it + 1);
  }
  asm volatile(".p2align 7");
  while (it < ntiles) {
    const int n0 = it * BN;
#pragma unroll
    for (int i = 0; i < DV / 32; i++) asm volatile("" : "+v"(o_acc[i]));  // (see fa_fwd_kernel.h: keeps O from being copied on every trip)
    wait_vmem();      // this wave's share of tile `it` is in LDS
    __syncthreads();  // so is everyone else's, and nobody still reads the other buffer
    if (it + 1 < ntiles) {
      stage(it + 1, buf ^ 1);
      if (it + 2 < ntiles) ask(it + 2);
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
    it++;
  }

  const float l_tot = half_sum(l_i);
  const float u_tot = kLse ? half_sum(u_i) : 0.f;
  if (p.n_splits > 1) {  // partial result of this split, fp32: [split][pair][row of nq_tiles * 128][D], m, l and u behind all of them
    if (mw + c < rows) {
      const int64_t all = (int64_t)p.c.B * p.c.HK * p.nq_tiles * kChunkRows, at = ((int64_t)b * p.c.HK + h) * p.nq_tiles * kChunkRows + mw + c;
      float* const op = p.part + (int64_t)split * all * (D + 3) + at * D;
      if (hf == 0) {
        float* const ml = p.part + (int64_t)split * all * (D + 3) + all * D + at * 3;
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

namespace {

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
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const PagedFwdParams p, int lanes) {
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

template <typename T, int D>
hipError_t launch_d(const PagedFwdParams& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.c.B * p.c.HK * p.nq_tiles;
  const int64_t pairs = (int64_t)p.c.B * p.c.HK;
  const dim3 grid((unsigned)(p.deal ? (pairs + 7) / 8 * 8 * p.nq_tiles : (items + 7) / 8 * 8), (unsigned)p.n_splits);
  if (p.lse) hipLaunchKernelGGL((fa_paged_chunk_kernel<T, D, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((fa_paged_chunk_kernel<T, D, false>), grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_splits <= 1) return e;
  const int lanes = join_lanes<D>(p.n_splits);
  const int64_t n = items * kChunkRows * kJoinCols<D> * lanes;
  hipLaunchKernelGGL((paged_chunk_join_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, lanes);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(const PagedFwdParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_d<T, 16>(p, stream);
    case 32: return launch_d<T, 32>(p, stream);
    case 64: return launch_d<T, 64>(p, stream);
    case 128: return launch_d<T, 128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_paged_chunk(const PagedFwdParams& p, int dtype, int head_dim, hipStream_t stream) {
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
