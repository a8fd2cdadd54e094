// fa_paged_key_weights: to the weight of every key of a paged cache is added what it receives of the new tokens' attention,
//   w[h, j] += sum over rows r of exp(scale q_r . k_j - lse_r)      (rows: the tokens and heads of the group, fa_paged_fwd.h)
// the probabilities formed again from the forward's lse: no second pass over V, no maxima.
//
// Two kernels.  Few rows (at most 32 a key head; a decode step): K streams past them, bound by HBM; waves stage 32-key tiles of their own as in
// fa_paged_decode.hip, over the same line of units.  Many: a workgroup takes one unit of that line (the launch's last ones find none), a wave owns 32 of its keys, their fragments in registers, and streams the rows past them in tiles of 64
// or 128 that the workgroup's four waves share through LDS; bound by vector instructions, three per 64 scores (4 sequences of 2000 .. 4001 keys, 8 key
// heads, 2 x 509 rows, d = 64: 26 us, vector instructions in 55 % of all SIMDs' cycles; one unit a workgroup by number instead of by the line 34, when this took
// 29.6, since a compute unit then has up to four workgroups of long sequences and another two).  Both form S = Q K^T, which leaves a key in a lane, so
// that its sum stays in the lane and has one owner.
#include <type_traits>

#include "fa_paged_line.h"

namespace fa {

namespace {

struct WeightsParams {
  PagedFwdParams f;
  uint32_t group_magic;  // ceil(2^32 / G), for numbers of at most 2^16: x / G = x * magic >> 32 (G = 1: not used)
};

template <int D, int BM_>
struct WCfg {
  static constexpr int BM = BM_;
  static constexpr int kTile = BM * D * 2;
  static constexpr int kRowOff = 2 * kTile;  // per buffer: BM lse, BM limits
  static constexpr int kRow = BM * 8;
  static constexpr int kLds = 2 * kTile + 2 * kRow;
};

}  // namespace

// (four waves a SIMD at least: with fewer the compiler puts the products into accumulation registers and moves them out one by one)
template <typename T, int D, int BM_>
__global__ void __launch_bounds__(256, 4) fa_paged_weights_kernel(const WeightsParams wp) {
  using C = WCfg<D, BM_>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  constexpr int CH = D / 8, BM = C::BM;
  const PagedFwdParams& p = wp.f;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[C::kLds];

  // Workgroups go to the eight XCDs in turn: each XCD takes a contiguous piece of the line of units, whose pairs' rows stay in its L2.
  const int sums0 = unit_sums(p.c, 0);
  const int64_t units = all_units(p.c, sums0), each = (units + 7) / 8;
  const int64_t u = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= each || u >= units) return;
  const Spot at_unit = spot_of(p.c, u, sums0);
  const int b = __builtin_amdgcn_readfirstlane(at_unit.b), h = __builtin_amdgcn_readfirstlane(at_unit.h), kblock = __builtin_amdgcn_readfirstlane(at_unit.unit);
  int q_begin = 0, Lq = 0;
  if (!paged_rows(p.c, b, &q_begin, &Lq)) return;
  const int Lk = paged_len(p.c, b), G = p.c.G, rows = Lq * G;
  if (kblock * 128 >= Lk) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const int key0 = kblock * 128 + wave * 32;  // of this wave
  const bool live = key0 < Lk;
  const float cs = p.scale_log2;
  const auto per_group = [&](int x) { return G == 1 ? x : (int)__umulhi((uint32_t)x, wp.group_magic); };

  // ---- this wave's keys (past the end: the last one, whose sum is not stored)
  const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
  const int key = key0 + c < Lk ? key0 + c : Lk - 1;
  vec8 kreg[D / 16];
  {
    const int g0 = key0 >> 4, last = (Lk - 1) >> 4;
    const int ga = g0 < last ? g0 : last, gb = g0 + 1 < last ? g0 + 1 : last;
    const char* const pa = p.c.k + page_of_group(p.c, table, ga) * p.c.k_ps + h * p.c.k_hs;
    const char* const pb = p.c.k + page_of_group(p.c, table, gb) * p.c.k_ps + h * p.c.k_hs;
    const int slot = key & ((1 << p.c.page_log2) - 1);
    const char* const at = ((key >> 4) == ga ? pa : pb) + slot * p.c.k_ss + hf * 16;
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) kreg[ks] = bitcast<vec8>(ld_global16(at + ks * 32));
  }

  // ---- rows: from the first that sees the workgroup's first key on
  const int past = Lk - Lq + 1;  // row r sees the keys below past + r / G
  int row_first = 0;
  if (p.causal) {
    const int tok = kblock * 128 - past + 1;
    row_first = tok > 0 ? tok * G : 0;
  }
  const int tile0 = row_first / BM, ntiles = (rows + BM - 1) / BM;
  // the first rows, as (token, head of the group), of the tile that is staged next and of the one whose lse and limits are asked for next
  int tok0 = __builtin_amdgcn_readfirstlane((tile0 * BM) / G), head0 = __builtin_amdgcn_readfirstlane(tile0 * BM - tok0 * G);
  int ask_tok = tok0, ask_head = head0;
  constexpr int RPI = 64 / CH;                        // rows per direct-to-LDS instruction
  constexpr int TI = BM / RPI;                        // instructions of a tile
  const int rl = lane / CH, pch = lane % CH;
  auto stage = [&](int it, int buf) {
    const char* const qb = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok0) * p.q_rs + (int64_t)h * G * p.q_hs);
#pragma unroll
    for (int i = 0; i < TI; i++) {
      if (TI >= 4 ? (i & 3) != wave : i != wave) continue;
      int r = i * RPI + rl;
      const int sw = tile_swz<D, kSwzRow>(r);
      const int most = rows - 1 - it * BM;
      r = r < most ? r : most;
      const int x = head0 + r, t = per_group(x), g = x - t * G;
      dma16(qb, (uint32_t)(t * p.q_rs * 2 + g * p.q_hs * 2) + 16u * (uint32_t)(pch ^ sw), lds_raw + buf * C::kTile + i * 1024);
    }
  };
  // a row's lse (in log2 units; +inf: no row, or one that sees nothing) and limit
  float lse_next = INFINITY;
  int limit_next = 0;
  auto fetch_row = [&](int it) {  // a thread a row
    const int r = it * BM + tid;
    lse_next = -INFINITY;
    limit_next = 0;
    if (tid < BM && r < rows) {
      const int x = ask_head + tid, t = per_group(x), g = x - t * G;
      lse_next = p.lse[((int64_t)b * p.c.H + h * G + g) * p.sq_r + ask_tok + t];
      limit_next = p.causal ? past + ask_tok + t : Lk;
    }
  };
  auto store_row = [&](int buf) {
    if (tid < BM) {
      reinterpret_cast<float*>(lds_raw + C::kRowOff + buf * C::kRow)[tid] = lse_next == -INFINITY ? INFINITY : lse_next * kLog2e;
      reinterpret_cast<int*>(lds_raw + C::kRowOff + buf * C::kRow + BM * 4)[tid] = limit_next;
    }
  };
  int first_tok = tok0;  // of the tile in hand
  auto advance = [&]() {
    const int x = ask_head + BM, t = __builtin_amdgcn_readfirstlane(per_group(x));
    tok0 = ask_tok;
    head0 = ask_head;
    ask_tok += t;
    ask_head = x - t * G;
  };
  int qoff[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ks++) qoff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);

  float sum[2] = {0.f, 0.f};
  int it = tile0, buf = 0;
  if (it < ntiles) {
    fetch_row(it);
    stage(it, 0);
    store_row(0);
    advance();
    fetch_row(it + 1);
    advance();
  }
  while (it < ntiles) {
    wait_vmem();
    __syncthreads();
    const int next_tok = tok0;
    if (it + 1 < ntiles) {
      store_row(buf ^ 1);
      stage(it + 1, buf ^ 1);
      fetch_row(it + 2);
      advance();
    }
    const int* const limits = reinterpret_cast<const int*>(lds_raw + C::kRowOff + buf * C::kRow + BM * 4);
    const float* const lses = reinterpret_cast<const float*>(lds_raw + C::kRowOff + buf * C::kRow);
    const T* const Qs = reinterpret_cast<const T*>(lds_raw + buf * C::kTile);
    if (live) {
      // d = 64: a half's exponentials in four groups, the next half's products between them, what either reads from LDS asked for a group before: a wave
      // alone on its SIMD does not wait for its chain of products (4 x 8 heads of 1024 keys, 2 x 1018 rows 33.7 -> 29.5 us; with four waves there 29.7 -> 29.5).
      // d = 128 has no registers for it, d = 32 loses a wave to it (22.7 -> 24.5).
      auto tile = [&](auto masked) {
        constexpr bool kBetween = D == 64;
        constexpr int KS = D / 16, NH = BM / 32;
        vec8 q[KS];
        f32x16 next;
        f32x4 l4;
        auto ask_q = [&](int half) {
#pragma unroll
          for (int ks = 0; ks < KS; ks++) q[ks] = *reinterpret_cast<const vec8*>(Qs + half * 32 * D + qoff[ks]);
        };
        auto ask_lse = [&](int group) { l4 = *reinterpret_cast<const f32x4*>(lses + 8 * group + 4 * hf); };
        auto products = [&](int ks0, int ks1) {
          if (ks0 == 0) {
#pragma unroll
            for (int r = 0; r < 16; r++) next[r] = 0.f;
          }
#pragma unroll
          for (int ks = ks0; ks < ks1; ks++) next = E::mfma32(q[ks], kreg[ks], next);
        };
        if (kBetween) {
          ask_q(0);
          ask_lse(0);
          products(0, KS);
          if (NH > 1) ask_q(1);
        }
#pragma unroll
        for (int half = 0; half < NH; half++) {
          if (!kBetween) {
#pragma unroll
            for (int r = 0; r < 16; r++) next[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) next = E::mfma32(*reinterpret_cast<const vec8*>(Qs + half * 32 * D + qoff[ks]), kreg[ks], next);
          }
          const f32x16 s = next;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (kBetween) {
              __builtin_amdgcn_sched_barrier(0);
              if (half + 1 < NH) products(j * KS / 4, (j + 1) * KS / 4);
              if (j == 3 && half + 2 < NH) ask_q(half + 2);
            } else {
              ask_lse(half * 4 + j);
            }
            const f32x4 lj = l4;
            if (kBetween && half * 4 + j + 1 < NH * 4) ask_lse(half * 4 + j + 1);
            f32x4 e;
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] = fast_exp2(__builtin_fmaf(s[4 * j + i], cs, -lj[i]));
            if constexpr (decltype(masked)::value) {
#pragma unroll
              for (int i = 0; i < 4; i++)
                if (key >= limits[half * 32 + 8 * j + 4 * hf + i]) e[i] = 0.f;
            }
            sum[j & 1] += (e[0] + e[1]) + (e[2] + e[3]);
          }
        }
      };
      // (whether the tile's first row does not see all of the wave's keys)
      if (p.causal && past + first_tok < key0 + 32) tile(std::true_type{});
      else tile(std::false_type{});
    }
    first_tok = next_tok;
    buf ^= 1;
    it++;
  }
  const float all = half_sum(sum[0] + sum[1]);
  if (hf == 0 && key0 + c < Lk) {
    const int page = table[key >> p.c.page_log2];
    if (page_is_one(page, p.c.n_pages)) {
      float* const w = p.c.weights + (((int64_t)page * p.c.HK + h) << p.c.page_log2) + (key & ((1 << p.c.page_log2) - 1));
      *w += all;
    }
  }
}

namespace {

template <int D>
struct FewCfg {
  static constexpr int NW = 4, BN = 32;
  static constexpr int kTile = BN * D * 2;
  static constexpr int kWave = 2 * kTile;      // two stages
  static constexpr int kKeys = 2048;           // keys whose sums wait in LDS to be added to the weights
  static constexpr int kLds = NW * kWave + kKeys * 4;
};
// Workgroups resident at once: 72 KB of LDS at d = 128, 40 at 64; below, as many as the waves fill the SIMDs with
constexpr int few_resident(int D) { return 256 * (D == 128 ? 2 : 4); }

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(256, D == 128 ? 2 : 4) fa_paged_weights_few_kernel(const PagedFwdParams p) {
  using C = FewCfg<D>;
  using E = Elem<T>;
  using vec8 = typename E::vec8;
  using Stager = GroupStager<D, kSwzRow>;
  constexpr int NW = C::NW, BN = C::BN, NI = 2 * Stager::NI;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[C::kLds];
  float* const sums = reinterpret_cast<float*>(lds_raw + NW * C::kWave);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const float cs = p.scale_log2;
  Stager st;
  st.init(lane, p.c.k_ss);
  unsigned char* const lds_wave = lds_raw + wave * C::kWave;
  int koff[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ks++) koff[ks] = frag_off<D, kSwzRow>(c, ks * 2 + hf);

  const int sums0 = unit_sums(p.c, 0);
  const int64_t units = all_units(p.c, sums0);
  const int n = sharers(p, units);
  if ((int)blockIdx.x >= n || units == 0) return;
  int64_t u = share_begin(units, blockIdx.x, n);
  const int64_t u_end = share_begin(units, blockIdx.x + 1, n);
  Spot at = spot_of(p.c, u, sums0);

  while (u < u_end) {
    const int b = __builtin_amdgcn_readfirstlane(at.b), h = __builtin_amdgcn_readfirstlane(at.h);
    const int unit0 = __builtin_amdgcn_readfirstlane(at.unit), pair_units = __builtin_amdgcn_readfirstlane(at.units);
    int unit1 = u_end - u < pair_units - unit0 ? unit0 + (int)(u_end - u) : pair_units;
    unit1 = unit1 - unit0 <= C::kKeys / kDecodeUnit ? unit1 : unit0 + C::kKeys / kDecodeUnit;
    // a tile's two groups of 16 keys: their pages are asked for a step before they are needed, those of the first two tiles together with the lengths
    const int32_t* const table = p.c.table + (int64_t)b * p.c.table_rs;
    const int k_lo = unit0 * kDecodeUnit;
    int page[2], page2[2];
    auto ask = [&](int t, int (&to)[2]) {
#pragma unroll
      for (int j = 0; j < 2; j++) to[j] = page_of_group(p.c, table, (k_lo >> 4) + 2 * t + j);
    };
    ask(wave, page);
    ask(wave + NW, page2);
    int q_begin = 0, Lq = 0;
    if (!paged_rows(p.c, b, &q_begin, &Lq)) return;  // (never: such a sequence has no units)
    const int Lk = paged_len(p.c, b), G = p.c.G, rows = Lq * G;
    const int k_hi = Lk < unit1 * kDecodeUnit ? Lk : unit1 * kDecodeUnit;
    const int ntiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
    const char* const kb = p.c.k + h * p.c.k_hs;
    const int last_group = (Lk - 1) >> 4;
    auto issue = [&](int t, int stage, const int (&pages)[2]) {
      const int g0 = (k_lo >> 4) + 2 * t;
      const bool both = g0 < last_group;  // (else the tile's second half repeats the last key, in the first one's page)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int g = both ? g0 + j : g0, pg = both ? pages[j] : pages[0];
        st.issue(kb + pg * p.c.k_ps + slot_of_group(p.c, g) * p.c.k_ss, p.c.k_ss, g < last_group ? 15 : (Lk - 1) & 15,
                 lds_wave + stage * C::kTile + j * Stager::kBytes);
      }
    };
    int t = wave, stage = 0;
    if (t < ntiles) issue(t, 0, page);
    if (t + NW < ntiles) issue(t + NW, 1, page2);
    // the rows: lane c holds row c's fragments; of the 16 that a lane's results belong to, lse (log2 units; +inf: no row, or one that sees nothing)
    // and limit.  Waited for here, with the first two tiles: the main loop counts this wave's outstanding loads.
    const int row = c < rows ? c : rows - 1, tok = row / G;
    vec8 qreg[D / 16];
    const T* const qp = reinterpret_cast<const T*>(p.q) + (int64_t)(q_begin + tok) * p.q_rs + (int64_t)(h * G + (row - tok * G)) * p.q_hs + hf * 8;
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) qreg[ks] = bitcast<vec8>(ld_global16(qp + ks * 16));
    float lse[16];
    int limit[16];
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int x = 8 * (r >> 2) + 4 * hf + (r & 3), xc = x < rows ? x : rows - 1, xt = xc / G;
      const float v = p.lse[((int64_t)b * p.c.H + h * G + (xc - xt * G)) * p.sq_r + xt];
      lse[r] = x >= rows || v == -INFINITY ? INFINITY : v * kLog2e;
      limit[r] = p.causal ? Lk - Lq + 1 + xt : Lk;
    }
    wait_vmcnt<0>();
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) asm volatile("" : "+v"(qreg[ks]));
#pragma unroll
    for (int r = 0; r < 16; r++) asm volatile("" : "+v"(lse[r]));
    const int least_limit = p.causal ? Lk - Lq + 1 : Lk;  // of row 0

    for (; t < ntiles; t += NW) {
      if (t + NW < ntiles) wait_vmcnt<NI>();  // (its NI loads were issued after this tile's)
      else wait_vmcnt<0>();
      if (t + 2 * NW < ntiles) ask(t + 2 * NW, page);
      const T* const Ks = reinterpret_cast<const T*>(lds_wave + stage * C::kTile);
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ks++) s = E::mfma32(qreg[ks], *reinterpret_cast<const vec8*>(Ks + koff[ks]), s);
      if (t + 2 * NW < ntiles) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the stage has been read before it is refilled
        issue(t + 2 * NW, stage, page);
      }
      const int key = k_lo + t * BN + c;
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = fast_exp2(__builtin_fmaf(s[r], cs, -lse[r]));
      if (k_lo + t * BN + BN > least_limit) {
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (key >= limit[r]) s[r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; r += 4) sum += (s[r] + s[r + 1]) + (s[r + 2] + s[r + 3]);
      sum = half_sum(sum);
      if (hf == 0) sums[t * BN + c] = sum;
      stage ^= 1;
    }
    __syncthreads();
    for (int i = tid; i < k_hi - k_lo; i += 64 * NW) {
      const int key = k_lo + i, pg = table[key >> p.c.page_log2];
      if (page_is_one(pg, p.c.n_pages)) {
        float* const w = p.c.weights + (((int64_t)pg * p.c.HK + h) << p.c.page_log2) + (key & ((1 << p.c.page_log2) - 1));
        *w += sums[i];
      }
    }
    u += unit1 - unit0;
    if (u >= u_end) return;
    if (unit1 < pair_units) at.unit = unit1;
    else if (!next_pair(p.c, &at)) return;  // (never: the line does not end here)
    __syncthreads();  // the sums have been read
  }
}

namespace {

template <typename T, int D>
hipError_t launch_d(const WeightsParams& p, hipStream_t stream) {
  const int64_t blocks = (int64_t)p.f.c.B * p.f.c.HK * ((p.f.c.max_keys + 127) / 128);
  if (blocks >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
  if (p.f.c.max_sq * p.f.c.G <= kDecodeMaxQ) {
    PagedFwdParams f = p.f;
    f.groups = (int)(blocks < few_resident(D) ? blocks : few_resident(D));  // (a block of 128 keys is a unit)
    hipLaunchKernelGGL((fa_paged_weights_few_kernel<T, D>), dim3((unsigned)f.groups), dim3(256), 0, stream, f);
  } else {
    // rows of a tile: work enough to cover the next one's loads, where there are as many (1 x 8 heads, 2 x 1000 rows, d = 64 30.4 us, in tiles of 64 32.9; d = 32 23.2, 26.7)
    constexpr int kMost = D == 128 ? 64 : 128;
    if (p.f.c.max_sq * p.f.c.G <= 64) hipLaunchKernelGGL((fa_paged_weights_kernel<T, D, 64>), dim3((unsigned)(blocks + 7) / 8 * 8), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((fa_paged_weights_kernel<T, D, kMost>), dim3((unsigned)(blocks + 7) / 8 * 8), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(const WeightsParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 16: return launch_d<T, 16>(p, stream);
    case 32: return launch_d<T, 32>(p, stream);
    case 64: return launch_d<T, 64>(p, stream);
    case 128: return launch_d<T, 128>(p, stream);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace

hipError_t launch_paged_key_weights(const PagedFwdParams& f, int dtype, int head_dim, hipStream_t stream) {
  WeightsParams p{f, f.c.G > 1 ? (uint32_t)((((uint64_t)1 << 32) + f.c.G - 1) / f.c.G) : 0u};
  return dtype == 0 ? launch_t<_Float16>(p, head_dim, stream) : launch_t<__bf16>(p, head_dim, stream);
}

}  // namespace fa
